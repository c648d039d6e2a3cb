// evict.hip -- eviction from a cache by accumulated attention weight.
//
// Every (row, head) of a paged cache holds n = len slots.  If n > budget, the `budget` slots stay
// that come first by (protected, weight descending, slot ascending); a slot is protected when its
// position is below `sinks` or among the `recent` highest (position >= max + 1 - recent).  A NaN
// weight counts as the lowest.  The i-th dropped slot below `budget` receives the row of the i-th
// kept slot at or past it, so that what stays lies in [0, budget): sources and destinations never
// overlap, every move is independent, and only the rows that must move do (one a head when a full
// cache took one token).  Weights and positions go to new arrays; the rows move in place.
//
// Kernel 1, one workgroup per (row, head): the budget-th best key by counting digits (keys are 32
// bits, larger is better), then one pass in slot order that numbers ties, holes and movers.
// Kernel 2 moves the rows.
#include "dgs_block.cuh"
#include "dgs_state.cuh"

namespace dgs {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMoveThreads = 256;
constexpr int kDigits = 2048;  // 11 bits: the sign, the exponent and two bits of the mantissa first

struct EvictArgs {
  EvictCall e;
  int64_t room;  // holes a (row, head) can have
  int32_t *moves;  // [rows * heads], the number of moves
  int32_t *holes, *movers;  // [rows * heads, room]
  GatherGuard gd;
};

// Larger is better; a protected slot beats every weight.
__device__ __forceinline__ uint32_t key_of(float w, bool fixed) {
  if (fixed) return 0xffffffffu;
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 ranks with 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int64_t evict_length(const EvictArgs &a, int64_t row, bool report) {
  const int64_t len = a.e.lens[row];
  const int64_t cap = a.e.width * a.e.page < a.e.cols ? a.e.width * a.e.page : a.e.cols;
  if ((uint64_t)len > (uint64_t)cap) {
    if (report) report_bad_id(a.gd.err, kAsyncErrLength, len, cap + 1, a.gd.tag);
    return len < 0 ? 0 : cap;
  }
  return len;
}

__global__ __launch_bounds__(kPlanThreads) void k_evict_plan(EvictArgs a) {
  __shared__ uint32_t s_hist[kDigits];
  __shared__ uint32_t s_scan[kPlanThreads / 64];
  __shared__ int32_t s_max[kPlanThreads / 64];
  __shared__ uint32_t s_digit, s_left;
  const EvictCall &e = a.e;
  const int64_t pair = blockIdx.x;
  const int64_t row = pair / e.heads;
  const int tid = threadIdx.x;
  const int64_t n = evict_length(a, row, tid == 0 && pair % e.heads == 0);
  const float *w = e.weights + pair * e.cols;
  const int32_t *pos = e.positions ? e.positions + pair * e.cols : nullptr;
  float *wo = e.weights_out + pair * e.cols;
  int32_t *po = e.positions_out + pair * e.cols;
  const int64_t keep = n < e.budget ? n : e.budget;
  if (tid == 0) {
    if (pair % e.heads == 0) {
      if (e.lens.bytes == 8)
        ((int64_t *)e.lens_out)[row] = keep;
      else
        ((int32_t *)e.lens_out)[row] = (int32_t)keep;
    }
    if (n <= e.budget) a.moves[pair] = 0;
  }
  for (int64_t j = keep + tid; j < e.cols; j += kPlanThreads) {
    wo[j] = 0.f;
    po[j] = -1;
  }
  if (n <= e.budget) {
    for (int64_t j = tid; j < n; j += kPlanThreads) {
      wo[j] = w[j];
      po[j] = pos ? pos[j] : (int32_t)j;
    }
    return;
  }
  // the highest position + 1
  int32_t top = -1;
  if (pos) {
    for (int64_t j = tid; j < n; j += kPlanThreads) top = pos[j] > top ? pos[j] : top;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const int32_t x = __shfl_xor(top, o, 64);
      top = x > top ? x : top;
    }
    if ((tid & 63) == 0) s_max[tid >> 6] = top;
    __syncthreads();
    for (int i = 0; i < kPlanThreads / 64; ++i) top = s_max[i] > top ? s_max[i] : top;
  } else {
    top = (int32_t)(n - 1);
  }
  const int64_t newest = (int64_t)top + 1 - e.recent;
  auto key_at = [&](int64_t j) {
    const int32_t p = pos ? pos[j] : (int32_t)j;
    return key_of(w[j], p < e.sinks || p >= newest);
  };
  // the keep-th largest key: digits of 11, 11 and 10 bits from the top
  uint32_t prefix = 0, left = (uint32_t)keep;
  int shift = 32;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    const uint32_t done = pass == 0 ? 0u : ~0u << shift;  // bits settled so far
    shift -= bits;
    for (int i = tid; i < kDigits; i += kPlanThreads) s_hist[i] = 0;
    __syncthreads();
    for (int64_t j = tid; j < n; j += kPlanThreads) {
      const uint32_t k = key_at(j);
      if ((k & done) == prefix) atomicAdd(&s_hist[(k >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // thread t owns digits 2047 - 2t and 2046 - 2t: an ascending scan counts from the largest
    const uint32_t hi = s_hist[kDigits - 1 - 2 * tid], lo = s_hist[kDigits - 2 - 2 * tid];
    uint32_t total;
    const uint32_t before = block_exclusive_scan<kPlanThreads>(hi + lo, &total, s_scan);
    if (before < left && left <= before + hi) {
      s_digit = kDigits - 1 - 2 * tid;
      s_left = left - before;
    } else if (before + hi < left && left <= before + hi + lo) {
      s_digit = kDigits - 2 - 2 * tid;
      s_left = left - before - hi;
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
    __syncthreads();
  }
  // In slot order: of the slots whose key equals the threshold the first `left` stay.
  int32_t *holes = a.holes + pair * a.room, *movers = a.movers + pair * a.room;
  uint32_t ties = 0, nh = 0, nm = 0;
  for (int64_t base = 0; base < n; base += kPlanThreads) {
    const int64_t j = base + tid;
    const bool in = j < n;
    const uint32_t k = in ? key_at(j) : 0u;
    const bool tie = in && k == prefix;
    uint32_t total;
    const uint32_t tr = block_exclusive_scan<kPlanThreads>(tie ? 1u : 0u, &total, s_scan) + ties;
    ties += total;
    const bool kept = in && (k > prefix || (tie && tr < left));
    const bool hole = in && !kept && j < e.budget, mover = kept && j >= e.budget;
    // both counts in one scan: fewer than 65536 of each in 1024 slots
    const uint32_t r = block_exclusive_scan<kPlanThreads>(
        (hole ? 1u : 0u) | (mover ? 0x10000u : 0u), &total, s_scan);
    if (hole) holes[nh + (r & 0xffffu)] = (int32_t)j;
    if (mover) movers[nm + (r >> 16)] = (int32_t)j;
    nh += total & 0xffffu;
    nm += total >> 16;
    if (kept && !mover) {
      wo[j] = w[j];
      po[j] = pos ? pos[j] : (int32_t)j;
    }
  }
  if (tid == 0) a.moves[pair] = (int32_t)nh;
  __threadfence_block();
  __syncthreads();
  for (uint32_t i = tid; i < nh; i += kPlanThreads) {
    const int32_t d = holes[i], s = movers[i];
    wo[d] = w[s];
    po[d] = pos ? pos[s] : s;
  }
}

template <int V>
struct MoveVec;
template <>
struct MoveVec<16> {
  using T = su32x4;
};
template <>
struct MoveVec<4> {
  using T = uint32_t;
};
template <>
struct MoveVec<1> {
  using T = uint8_t;
};

__device__ __forceinline__ int64_t store_slot(const EvictArgs &a, int64_t row, int64_t h,
                                              int32_t j) {
  const int64_t page = a.e.table[row * a.e.width + j / a.e.page];
  if ((uint64_t)page >= (uint64_t)a.e.pages) {
    report_bad_id(a.gd.err, kAsyncErrSlot, page, a.e.pages, a.gd.tag);
    return -1;
  }
  return (page * a.e.heads + h) * a.e.page + j % a.e.page;
}

// One wave per move.
template <int V>
__global__ __launch_bounds__(kMoveThreads) void k_evict_move(EvictArgs a, EvictStore store) {
  using T = typename MoveVec<V>::T;
  const int64_t pair = blockIdx.x;
  const int64_t row = pair / a.e.heads, h = pair % a.e.heads;
  const int moves = a.moves[pair];
  const int lane = threadIdx.x & 63;
  const int wave = blockIdx.y * (kMoveThreads / 64) + (threadIdx.x >> 6);
  const int waves = gridDim.y * (kMoveThreads / 64);
  const int64_t vecs = store.row_bytes / V;
  for (int i = wave; i < moves; i += waves) {
    const int64_t d = store_slot(a, row, h, a.holes[pair * a.room + i]);
    const int64_t s = store_slot(a, row, h, a.movers[pair * a.room + i]);
    if (d < 0 || s < 0) continue;
    T *dst = (T *)(store.p + d * store.row_bytes);
    const T *src = (const T *)(store.p + s * store.row_bytes);
    for (int64_t v = lane; v < vecs; v += 64) dst[v] = src[v];
  }
}

int64_t evict_room(const EvictCall &e) {
  const int64_t over = e.cols - e.budget;
  return over <= 0 ? 0 : (over < e.budget ? over : e.budget);
}
int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

}  // namespace

int64_t evict_workspace(const EvictCall &e) {
  const int64_t pairs = e.rows * e.heads;
  return up256(pairs * 4) + 2 * up256(pairs * evict_room(e) * 4);
}

void evict_rows(const EvictCall &e, void *ws, int64_t ws_bytes, hipStream_t st) {
  const int64_t pairs = e.rows * e.heads;
  if (pairs <= 0) return;
  DGS_CHECK(ws && ws_bytes >= evict_workspace(e), "evict: workspace too small");
  DGS_CHECK(pairs < (int64_t(1) << 31) && e.cols < (int64_t(1) << 30),
            "evict: too many rows or columns");
  EvictArgs a{};
  a.e = e;
  a.room = evict_room(e);
  char *w = static_cast<char *>(ws);
  a.moves = (int32_t *)w;
  a.holes = (int32_t *)(w + up256(pairs * 4));
  a.movers = (int32_t *)(w + up256(pairs * 4) + up256(pairs * a.room * 4));
  a.gd = state_guard(kAsyncErrSlot, e.pages);
  k_evict_plan<<<(unsigned)pairs, kPlanThreads, 0, st>>>(a);
  DGS_LAUNCH_CHECK();
  if (a.room == 0) return;
  int64_t ny = ceil_div(a.room, 32);
  const int64_t fill = ceil_div(8192, pairs);
  if (ny > fill) ny = fill;
  if (ny > 1024) ny = 1024;
  const dim3 grid((unsigned)pairs, (unsigned)ny);
  for (int i = 0; i < e.nstores; ++i) {
    const EvictStore &s = e.stores[i];
    const uintptr_t al = (uintptr_t)s.p | (uintptr_t)s.row_bytes;
    if (al % 16 == 0)
      k_evict_move<16><<<grid, kMoveThreads, 0, st>>>(a, s);
    else if (al % 4 == 0)
      k_evict_move<4><<<grid, kMoveThreads, 0, st>>>(a, s);
    else
      k_evict_move<1><<<grid, kMoveThreads, 0, st>>>(a, s);
    DGS_LAUNCH_CHECK();
  }
}

}  // namespace dgs
