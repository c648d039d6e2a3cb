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
// The plan, one workgroup per (row, head): weights and positions are read once, four slots a load,
// and stay in registers as keys (32 bits, larger is better; rows past 32768 slots read them again
// each time); the budget-th best key by counting digits; then ties, holes and movers are numbered
// in slot order by scans over lanes and waves.  What lies below the budget is copied as it passes and the
// holes are overwritten afterwards.  16 rows of 8 heads of 20000 to 32768 slots to 4096: 34 us, more than half
// of which its waves wait (profiles/state_cache_counters.txt); a workgroup a (row, head) leaves half of the
// card idle there.
// The moves are a kernel of their own, over all stores; where there can only be a few (a cache
// that takes single tokens) the plan's workgroup does them.
#include "dgs_block.cuh"
#include "dgs_state.cuh"

namespace dgs {
namespace {

constexpr int kMoveThreads = 256;
constexpr int kDigits = 2048;  // 11 bits: the sign, the exponent and two bits of the mantissa first
// Moves a (row, head) can have at most for its plan's workgroup to do them.  64 rows of 8 heads of 4000
// to 4097 slots, 256 bytes a row, room 237: 40 us, 43 with a kernel for the moves; one such row 24.6, 24.1;
// 33 rows of 2 heads of 200 slots, room 100: 14, 18; room 500: 20 to 29 us in the plan, 18 apart.
constexpr int kFewMoves = 256;
static_assert(kFewMoves >= 128, "rows of 256 slots have at most 128 moves");

struct EvictArgs {
  EvictCall e;
  int64_t room;  // holes a (row, head) can have
  int32_t *moves;  // [rows * heads], the number of moves
  int32_t *holes, *movers;  // [rows * heads, room]
  StateGuard gd;
};

// Inclusive sum over the lanes of a wave by lane moves: within rows of 16, then the rows' last lanes.
__device__ __forceinline__ uint32_t lanes_before_and_me(uint32_t x) {
  auto add = [&](auto moved) { x += (uint32_t)moved; };
  add(__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false));  // row_shr 1
  add(__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
  add(__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));  // lane 15 of rows 0, 2 to 1, 3
  add(__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));  // lane 31 to rows 2, 3
  return x;
}

// Larger is better; a protected slot beats every weight.  Positions that repeat can protect more slots
// than stay: the threshold comes out as kFixed then, and the selection is made once more with
// protected_key, which ranks them by weight and puts all others behind.
constexpr uint32_t kFixed = 0xffffffffu;
__device__ __forceinline__ uint32_t key_of(float w, bool fixed) {
  if (fixed) return kFixed;
  if (w != w) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.f);  // -0 ranks with 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t protected_key(float w, bool fixed) {
  return fixed ? key_of(w, false) : 0u;
}

__device__ __forceinline__ int evict_length(const EvictArgs &a, int64_t row, bool report) {
  const int64_t len = a.e.lens[row];
  const int64_t room = a.e.width * a.e.page, cap = room < a.e.cols ? room : a.e.cols;
  if ((uint64_t)len > (uint64_t)cap) {
    if (report) report_bad_id(a.gd.err, kAsyncErrLength, len, cap + 1, a.gd.tag);
    return len < 0 ? 0 : (int)cap;
  }
  return (int)len;
}

__device__ __forceinline__ int64_t store_slot(const EvictArgs &a, int64_t row, int h, uint32_t j) {
  const uint32_t size = (uint32_t)a.e.page, p = j / size;
  const int64_t page = a.e.table[row * a.e.width + p];
  if ((uint64_t)page >= (uint64_t)a.e.pages) {
    report_bad_id(a.gd.err, kAsyncErrSlot, page, a.e.pages, a.gd.tag);
    return -1;
  }
  return (page * a.e.heads + h) * a.e.page + (j - p * size);
}

// kU rows at a time from source to destination slots (negative: none), by 1 << lg lanes each.
template <typename T, int kU>
__device__ __forceinline__ void move_rows(const EvictStore &st, const int64_t (&s)[kU],
                                          const int64_t (&d)[kU], int sub, int lg) {
  const int64_t vecs = st.row_bytes / sizeof(T);
  for (int64_t v = sub; v < vecs; v += 1 << lg) {
    T x[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u)
      x[u] = ((const T *)(st.p + (s[u] < 0 ? 0 : s[u]) * st.row_bytes))[v];
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (s[u] >= 0) ((T *)(st.p + d[u] * st.row_bytes))[v] = x[u];
  }
}
template <int kU>
__device__ __forceinline__ void move_store(const EvictStore &st, const int64_t (&s)[kU],
                                           const int64_t (&d)[kU], int sub, int lg) {
  const uintptr_t al = (uintptr_t)st.p | (uintptr_t)st.row_bytes;
  if (al % 16 == 0)
    move_rows<su32x4, kU>(st, s, d, sub, lg);
  else if (al % 4 == 0)
    move_rows<uint32_t, kU>(st, s, d, sub, lg);
  else
    move_rows<uint8_t, kU>(st, s, d, sub, lg);
}

// Moves first, first + stride, ... of a (row, head)'s list in one store, kU at a time.
template <int kU>
__device__ __forceinline__ void move_list(const EvictArgs &a, const EvictStore &st, int64_t row,
                                          int h, const int32_t *holes, const int32_t *movers,
                                          int moves, int first, int stride, int sub, int lg) {
  for (int i = first; i < moves; i += kU * stride) {
    int64_t d[kU], s[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const bool in = i + u * stride < moves;
      const int x = in ? i + u * stride : i;
      d[u] = store_slot(a, row, h, holes[x]);
      s[u] = store_slot(a, row, h, movers[x]);
      if (!in || d[u] < 0) s[u] = -1;
    }
    move_store<kU>(st, s, d, sub, lg);
  }
}
// 1 << lg lanes for a row: one for each 16 bytes, up to a wave.
__device__ __forceinline__ int row_lanes(const EvictStore &st, int lg) {
  while (lg < 6 && (16 << lg) < st.row_bytes) ++lg;
  return lg;
}

// What the plans share: the row's sizes, the slots that no eviction touches, its outputs.
struct PlanRow {
  int64_t pair, row;
  int h, n, cols, budget, keep;
  const float *w;
  const int32_t *pos;
  float *wo;
  int32_t *po;
};
__device__ __forceinline__ PlanRow plan_row(const EvictArgs &a) {
  const EvictCall &e = a.e;
  PlanRow r;
  r.pair = blockIdx.x;
  r.row = r.pair / e.heads;
  r.h = (int)(r.pair % e.heads);
  r.n = evict_length(a, r.row, threadIdx.x == 0 && r.h == 0);
  r.cols = (int)e.cols;
  r.w = e.weights + r.pair * e.cols;
  r.pos = e.positions ? e.positions + r.pair * e.cols : nullptr;
  r.wo = e.weights_out + r.pair * e.cols;
  r.po = e.positions_out + r.pair * e.cols;
  r.budget = (int)(e.budget < r.cols ? e.budget : r.cols);
  r.keep = r.n < r.budget ? r.n : r.budget;
  if (threadIdx.x == 0) {
    if (r.h == 0) {
      if (e.lens.bytes == 8)
        ((int64_t *)e.lens_out)[r.row] = r.keep;
      else
        ((int32_t *)e.lens_out)[r.row] = r.keep;
    }
    if (a.moves && r.n <= r.budget) a.moves[r.pair] = 0;
  }
  return r;
}
// The largest x of the workgroup (barrier inside).
template <int THREADS>
__device__ __forceinline__ int32_t block_max(int32_t x, int32_t *lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const int32_t y = __shfl_xor(x, o, 64);
    x = y > x ? y : x;
  }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) x = lds[i] > x ? lds[i] : x;
  return x;
}
// The digit that holds the `left`-th largest key of the histogram; left becomes its rank there,
// found[2] the keys there.
template <int THREADS>
__device__ __forceinline__ uint32_t pick_digit(const uint32_t *hist, uint32_t &left, uint32_t *scan,
                                               uint32_t *found) {
  constexpr int kOwn = kDigits / THREADS;
  // thread t owns kOwn digits counted from the largest: an ascending scan of them
  constexpr int kWaves = THREADS / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t mine[kOwn], sum = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    mine[i] = hist[kDigits - 1 - ((int)threadIdx.x * kOwn + i)];
    sum += mine[i];
  }
  const uint32_t upto = lanes_before_and_me(sum);
  if (lane == 63) scan[wave] = upto;
  __syncthreads();
  uint32_t before = upto - sum;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) before += v < wave ? scan[v] : 0u;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    if (before < left && left <= before + mine[i]) {
      found[0] = kDigits - 1 - ((int)threadIdx.x * kOwn + i);
      found[1] = left - before;
      found[2] = mine[i];
    }
    before += mine[i];
  }
  __syncthreads();
  left = found[1];
  return found[0];
}
// Weights and positions of the slots that take a mover's row, and with FUSED the rows.  (Taken along by
// the kernel that moves rows they cost it 15 us and spare 2 here: 435 thousand moves of two stores of
// 256 bytes a row.)
template <int THREADS, bool FUSED>
__device__ __forceinline__ void plan_end(const EvictArgs &a, const PlanRow &r,
                                         const int32_t *holes, const int32_t *movers,
                                         uint32_t all) {
  if (!FUSED && threadIdx.x == 0) a.moves[r.pair] = (int32_t)all;
  __syncthreads();  // the lists and the copies are written: a workgroup sees its stores past a barrier
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < all; i += THREADS) {
    const int32_t d = holes[i], s = movers[i];
    r.wo[d] = r.w[s];
    r.po[d] = r.pos ? r.pos[s] : s;
  }
  if (FUSED && a.e.nstores > 0) {
    // the stores side by side, as many lanes a row as the longest has 16-byte pieces
    int lg = 0;
    for (int st = 0; st < a.e.nstores; ++st) lg = row_lanes(a.e.stores[st], lg);
    const int sub = threadIdx.x & ((1 << lg) - 1), group = threadIdx.x >> lg;
    const int groups = THREADS >> lg, per = groups > a.e.nstores ? groups / a.e.nstores : 1;
    const int first = group % per;
    for (int st = group / per; st < a.e.nstores; st += groups / per) {
      const EvictStore &to = a.e.stores[st];
      if ((int)all <= per)
        move_list<1>(a, to, r.row, r.h, holes, movers, (int)all, first, per, sub, lg);
      else
        move_list<4>(a, to, r.row, r.h, holes, movers, (int)all, first, per, sub, lg);
    }
  }
}

// Rows of at most THREADS slots, one a thread: a slot stays if fewer than `keep` come before it, and
// every thread counts them.  33 rows of 2 heads of 0 to 77 slots: 9.1 us, 13.6 with digits and one move a
// wave at a time: a chain of loads (length, table, row), bound by nothing else.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_evict_plan_small(EvictArgs a) {
  constexpr int kWaves = THREADS / 64;
  __shared__ uint32_t s_key[THREADS], s_run[kWaves], s_fixed[kWaves];
  __shared__ int32_t s_max[kWaves];
  __shared__ int32_t s_hole[THREADS / 2], s_mover[THREADS / 2];  // as many of one as of the other
  const int j = threadIdx.x, lane = j & 63, wave = j >> 6;
  const int64_t at = blockIdx.x * a.e.cols + j;
  const bool in = j < a.e.cols;  // a row may have no columns, and the arrays no memory
  const float w = in ? a.e.weights[at] : 0.f;
  const int32_t p = in && a.e.positions ? a.e.positions[at] : j;
  const PlanRow r = plan_row(a);
  if (j < r.cols) {
    r.wo[j] = j < r.keep ? w : 0.f;
    r.po[j] = j < r.keep ? p : -1;
  }
  if (r.n <= r.budget) return;
  const int32_t top = block_max<THREADS>(j < r.n ? p : -1, s_max);
  const int64_t newest = (int64_t)top + 1 - a.e.recent;
  const bool fixed = j < r.n && (p < a.e.sinks || p >= newest);
  // past the row: 0, behind every key
  uint32_t key = j < r.n ? key_of(w, fixed) : 0u;
  s_key[j] = key;
  const uint64_t all_fixed = __ballot(fixed);
  if (lane == 0) s_fixed[wave] = __popcll(all_fixed);
  __syncthreads();
  uint32_t held = 0;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) held += s_fixed[v];
  if (held > (uint32_t)r.keep) {
    key = protected_key(w, fixed);
    s_key[j] = key;  // a thread's own: the others read it past the barrier
    __syncthreads();
  }
  // of equal keys the lower slot comes first
  int before = 0;
  for (int v = 0; v < kWaves; ++v) {
    if (v * 64 >= r.n) break;
    if (v == wave) {
#pragma unroll 16
      for (int i = 0; i < 64; ++i) {
        const uint32_t k = s_key[v * 64 + i];
        before += k > key || (k == key && i < lane);
      }
    } else {
      const uint32_t least = v < wave ? key - (key != 0) : key;
#pragma unroll 16
      for (int i = 0; i < 64; ++i) before += s_key[v * 64 + i] > least;
    }
  }
  const bool kept = j < r.n && before < r.keep;
  const bool hole = j < r.budget && !kept, mover = j >= r.budget && kept;
  // as many movers as holes: both numbers in a word
  const uint32_t own = (hole ? 1u : 0u) | (mover ? 0x10000u : 0u);
  const uint32_t sum = lanes_before_and_me(own);
  if (lane == 63) s_run[wave] = sum;
  __syncthreads();
  uint32_t rank = sum - own, all = 0;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    if (v < wave) rank += s_run[v];
    all += s_run[v];
  }
  if (hole) s_hole[rank & 0xffffu] = j;
  if (mover) s_mover[rank >> 16] = j;
  plan_end<THREADS, true>(a, r, s_hole, s_mover, all & 0xffffu);
}

// The selection where every step reads weights and positions again: the threshold by digits, then ties,
// holes and movers in slot order, of which a wave takes a run of n / kWaves slots.  Returns the moves.
// s_cnt: 3 kWaves words.
template <int THREADS>
__device__ __forceinline__ uint32_t plan_again(const EvictArgs &a, const PlanRow &r, int64_t newest,
                                               bool only_protected, int32_t *holes, int32_t *movers,
                                               uint32_t *s_hist, uint32_t *s_scan, uint32_t *s_found,
                                               uint32_t *s_cnt) {
  constexpr int kWaves = THREADS / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = r.n;
  auto key_at = [&](int j) {
    const int32_t p = r.pos ? r.pos[j] : j;
    const bool fixed = p < a.e.sinks || p >= newest;
    return only_protected ? protected_key(r.w[j], fixed) : key_of(r.w[j], fixed);
  };
  uint32_t prefix, left;
#pragma unroll 1
  while (true) {
    prefix = 0;
    left = (uint32_t)r.keep;
    int shift = 32;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10;
      const uint32_t done = pass == 0 ? 0u : ~0u << shift;
      shift -= bits;
      for (int i = tid; i < kDigits; i += THREADS) s_hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int j = tid; j < n; j += THREADS) {
        const uint32_t k = key_at(j);
        if ((k & done) == prefix) atomicAdd(&s_hist[(k >> shift) & ((1u << bits) - 1)], 1u);
      }
      __syncthreads();
      prefix |= pick_digit<THREADS>(s_hist, left, s_scan, s_found) << shift;
    }
    if (prefix != kFixed || s_found[2] == left) break;
    only_protected = true;
  }
  const int seg = ((n + kWaves - 1) / kWaves + 63) & ~63;
  const int j0 = wave * seg, j1 = j0 + seg < n ? j0 + seg : n;
  const uint64_t below = lane == 0 ? 0ull : ~0ull >> (64 - lane);
  auto before_wave = [&](const uint32_t *c) {
    uint32_t s = 0;
    for (int i = 0; i < wave; ++i) s += c[i];
    return s;
  };
  uint32_t cnt = 0;
  for (int b = j0; b < j1; b += 64)
    cnt += __popcll(__ballot(b + lane < j1 && key_at(b + lane) == prefix));
  if (lane == 0) s_cnt[wave] = cnt;
  __syncthreads();
  const uint32_t tie0 = before_wave(s_cnt);
  uint32_t nh = 0, nm = 0;
  for (int turn = 0; turn < 2; ++turn) {  // count, then write
    uint32_t ties = tie0;
    for (int b = j0; b < j1; b += 64) {
      const int j = b + lane;
      const bool in = j < j1;
      const uint32_t k = key_at(in ? j : j1 - 1);
      const bool tie = in && k == prefix;
      const uint64_t tb = __ballot(tie);
      const bool kept = in && (k > prefix || (tie && ties + __popcll(tb & below) < left));
      ties += __popcll(tb);
      const uint64_t hb = __ballot(in && !kept && j < r.budget);
      const uint64_t mb = __ballot(kept && j >= r.budget);
      if (turn == 1) {
        if ((hb >> lane) & 1) holes[nh + __popcll(hb & below)] = j;
        if ((mb >> lane) & 1) movers[nm + __popcll(mb & below)] = j;
      }
      nh += __popcll(hb);
      nm += __popcll(mb);
    }
    if (turn == 0) {
      if (lane == 0) {
        s_cnt[kWaves + wave] = nh;
        s_cnt[2 * kWaves + wave] = nm;
      }
      __syncthreads();
      nh = before_wave(s_cnt + kWaves);
      nm = before_wave(s_cnt + 2 * kWaves);
    }
  }
  uint32_t all = 0;
  for (int i = 0; i < kWaves; ++i) all += s_cnt[kWaves + i];
  return all;
}

// Rows of at most THREADS * kVecs * 4 slots: slot (v THREADS + t) 4 + i is thread t's.  ALIGNED:
// every row of weights and positions starts at 16 bytes.  Where one slot too many is held, as
// after every token of a full cache, the digits are not counted: the lowest key goes (of equal ones
// the last), one exchange over the workgroup.
template <int THREADS, int kVecs, bool FUSED, bool ALIGNED>
__global__ __launch_bounds__(THREADS) void k_evict_plan(EvictArgs a) {
  constexpr int kWaves = THREADS / 64, kRuns = kVecs * kWaves;  // a run: a wave's 256 slots of a v
  static_assert(kRuns <= 128, "one wave scans the runs, two a lane");
  __shared__ uint32_t s_hist[3][kDigits];
  __shared__ uint32_t s_scan[kWaves], s_found[3], s_run[kRuns];
  __shared__ int32_t s_max[kWaves];
  __shared__ uint64_t s_low[kWaves];
  __shared__ int32_t s_list[2 * kFewMoves];  // FUSED: holes, movers
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t key[kVecs][4];
  int32_t p[kVecs][4], top = -1;
  {
    // whole rows of the arrays, while the length is on its way
    const float *w = a.e.weights + blockIdx.x * a.e.cols;
    const int32_t *pos = a.e.positions ? a.e.positions + blockIdx.x * a.e.cols : nullptr;
    const int cols = (int)a.e.cols;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const int j = (v * THREADS + tid) * 4;
      if (v * THREADS * 4 >= cols) break;
      if (ALIGNED) {
        const int x = j < cols ? j : 0;
        *(su32x4 *)key[v] = *(const su32x4 *)(w + x);
        if (pos) *(su32x4 *)p[v] = *(const su32x4 *)(pos + x);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int x = j + i < cols ? j + i : 0;
          key[v][i] = __float_as_uint(w[x]);
          if (pos) p[v][i] = pos[x];
        }
      }
    }
  }
  for (int i = tid; i < 3 * kDigits; i += THREADS) (&s_hist[0][0])[i] = 0;
  const PlanRow r = plan_row(a);
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int j = (v * THREADS + tid) * 4;
    if (v * THREADS * 4 >= r.cols) break;
    if (!r.pos)
#pragma unroll
      for (int i = 0; i < 4; ++i) p[v][i] = j + i;
    su32x4 wo, po;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wo[i] = j + i < r.keep ? key[v][i] : 0u;
      po[i] = j + i < r.keep ? (uint32_t)p[v][i] : ~0u;
    }
    if (ALIGNED) {  // whole pieces of four
      if (j < r.cols) {
        *(su32x4 *)(r.wo + j) = wo;
        *(su32x4 *)(r.po + j) = po;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i < r.cols) {
          r.wo[j + i] = __uint_as_float(wo[i]);
          r.po[j + i] = (int32_t)po[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i < r.n && p[v][i] > top) top = p[v][i];
  }
  if (r.n <= r.budget) return;
  top = block_max<THREADS>(top, s_max);
  const int64_t newest = (int64_t)top + 1 - a.e.recent;
#pragma unroll
  for (int v = 0; v < kVecs; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      key[v][i] = key_of(__uint_as_float(key[v][i]), p[v][i] < a.e.sinks || p[v][i] >= newest);
  int32_t *holes = FUSED ? s_list : a.holes + r.pair * a.room;
  int32_t *movers = FUSED ? s_list + kFewMoves : a.movers + r.pair * a.room;
  // more protected slots than stay: rare, and not worth the registers
  auto rank_protected = [&]() {
    const uint32_t all = plan_again<THREADS>(a, r, newest, true, holes, movers, s_hist[0], s_scan, s_found,
                                             s_hist[1]);
    plan_end<THREADS, FUSED>(a, r, holes, movers, all);
  };
  if (r.n == r.budget + 1) {
    uint64_t low = ~0ull;  // key, then the complement of the slot
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = (v * THREADS + tid) * 4 + i;
        const uint64_t x = (uint64_t)key[v][i] << 32 | ~(uint32_t)j;
        if (j < r.n && x < low) low = x;
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t x = __shfl_xor((unsigned long long)low, o, 64);
      low = x < low ? x : low;
    }
    if (lane == 0) s_low[wave] = low;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) low = s_low[i] < low ? s_low[i] : low;
    if ((uint32_t)(low >> 32) == kFixed) return rank_protected();
    const int drop = (int)~(uint32_t)low;
    if (tid == 0) {
      holes[0] = drop;
      movers[0] = r.budget;
    }
    plan_end<THREADS, FUSED>(a, r, holes, movers, drop < r.budget ? 1u : 0u);
    return;
  }
  // the keep-th largest key: digits of 11, 11 and 10 bits from the top
  uint32_t prefix = 0, left = (uint32_t)r.keep;
  int shift = 32;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    const uint32_t done = pass == 0 ? 0u : ~0u << shift;  // bits settled so far
    shift -= bits;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      if (v * THREADS * 4 >= r.n) break;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t k = key[v][i];
        if ((v * THREADS + tid) * 4 + i < r.n && (k & done) == prefix)
          atomicAdd(&s_hist[pass][(k >> shift) & ((1u << bits) - 1)], 1u);
      }
    }
    __syncthreads();
    prefix |= pick_digit<THREADS>(s_hist[pass], left, s_scan, s_found) << shift;
  }
  if (prefix == kFixed && s_found[2] != left) return rank_protected();  // pick_digit ends in a barrier
  // Exclusive sums of the runs' counts in slot order (run = v, wave), in place.
  auto scan_runs = [&]() {
    __syncthreads();
    if (wave == 0) {
      const uint32_t x = 2 * lane < kRuns ? s_run[2 * lane] : 0u;
      const uint32_t y = 2 * lane + 1 < kRuns ? s_run[2 * lane + 1] : 0u;
      const uint32_t before = lanes_before_and_me(x + y) - x - y;
      if (2 * lane < kRuns) s_run[2 * lane] = before;
      if (2 * lane + 1 < kRuns) s_run[2 * lane + 1] = before + x;
      if (lane == 63) s_found[0] = before + x + y;
    }
    __syncthreads();
  };
  uint32_t kept = 0;  // bit 4 v + i
  const bool all_ties = s_found[2] == left;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    if (v * THREADS * 4 >= r.n) break;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = (v * THREADS + tid) * 4 + i < r.n;
      if (in && (key[v][i] > prefix || (all_ties && key[v][i] == prefix)))
        kept |= 1u << (4 * v + i);
    }
  }
  if (!all_ties) {
    // of the slots whose key equals the threshold the first `left` in slot order stay
    uint32_t tie = 0, at[kVecs];
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = (v * THREADS + tid) * 4 + i < r.n;
        if (in && key[v][i] == prefix) tie |= 1u << (4 * v + i);
      }
      const uint32_t own = __popc((tie >> (4 * v)) & 15u), sum = lanes_before_and_me(own);
      at[v] = sum - own;
      if (lane == 63) s_run[v * kWaves + wave] = sum;
    }
    scan_runs();
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      uint32_t rank = s_run[v * kWaves + wave] + at[v];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if ((tie >> (4 * v + i)) & 1) {
          if (rank < left) kept |= 1u << (4 * v + i);
          ++rank;
        }
    }
    __syncthreads();  // s_run is written again
  }
  // holes (dropped below the budget) in the low half, movers (kept at or past it) in the high one:
  // at most 32768 of each
  uint32_t hole = 0, mover = 0, at[kVecs];
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = (v * THREADS + tid) * 4 + i;
      const bool k = (kept >> (4 * v + i)) & 1;
      if (j < r.budget && !k) hole |= 1u << (4 * v + i);
      if (j >= r.budget && k) mover |= 1u << (4 * v + i);
    }
    const uint32_t own = __popc((hole >> (4 * v)) & 15u) | __popc((mover >> (4 * v)) & 15u) << 16;
    const uint32_t sum = lanes_before_and_me(own);
    at[v] = sum - own;
    if (lane == 63) s_run[v * kWaves + wave] = sum;
  }
  scan_runs();
  const uint32_t all = s_found[0] & 0xffffu;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    uint32_t rank = s_run[v * kWaves + wave] + at[v];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = (v * THREADS + tid) * 4 + i;
      if ((hole >> (4 * v + i)) & 1) holes[rank++ & 0xffffu] = j;
      if ((mover >> (4 * v + i)) & 1) {
        movers[rank >> 16] = j;
        rank += 0x10000u;
      }
    }
  }
  plan_end<THREADS, FUSED>(a, r, holes, movers, all);
}

// Longer rows.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_evict_plan_long(EvictArgs a) {
  constexpr int kWaves = THREADS / 64;
  __shared__ uint32_t s_hist[kDigits];
  __shared__ uint32_t s_scan[kWaves], s_found[3], s_cnt[3 * kWaves];
  __shared__ int32_t s_max[kWaves];
  const PlanRow r = plan_row(a);
  const int tid = threadIdx.x, n = r.n;
  for (int j = r.keep + tid; j < r.cols; j += THREADS) {
    r.wo[j] = 0.f;
    r.po[j] = -1;
  }
  int32_t top = -1;
#pragma unroll 4
  for (int j = tid; j < n; j += THREADS) {
    const int32_t p = r.pos ? r.pos[j] : j;
    if (j < r.keep) {
      r.wo[j] = r.w[j];
      r.po[j] = p;
    }
    top = p > top ? p : top;
  }
  if (n <= r.budget) return;
  top = block_max<THREADS>(top, s_max);
  const int64_t newest = (int64_t)top + 1 - a.e.recent;
  int32_t *holes = a.holes + r.pair * a.room, *movers = a.movers + r.pair * a.room;
  const uint32_t all = plan_again<THREADS>(a, r, newest, false, holes, movers, s_hist, s_scan, s_found, s_cnt);
  plan_end<THREADS, false>(a, r, holes, movers, all);
}

// Block (x, y, z): (row, head), a share of its moves, a store.  435 thousand moves of two stores of 256
// bytes a row (446 MB): 90 us, 5.0 TB/s.
__global__ __launch_bounds__(kMoveThreads) void k_evict_move(EvictArgs a) {
  const int64_t pair = blockIdx.x;
  const EvictStore &st = a.e.stores[blockIdx.z];
  const int lg = row_lanes(st, 0), groups = kMoveThreads >> lg;
  move_list<4>(a, st, pair / a.e.heads, (int)(pair % a.e.heads), a.holes + pair * a.room,
            a.movers + pair * a.room, a.moves[pair], blockIdx.y * groups + (threadIdx.x >> lg),
            groups * gridDim.y, threadIdx.x & ((1 << lg) - 1), lg);
}

int64_t evict_room(const EvictCall &e) {
  const int64_t over = e.cols - e.budget;
  return over <= 0 ? 0 : (over < e.budget ? over : e.budget);
}
int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

template <int THREADS, int kVecs, bool FUSED>
void launch_plan(const EvictArgs &a, hipStream_t st) {
  const unsigned pairs = (unsigned)(a.e.rows * a.e.heads);
  const uintptr_t at = (uintptr_t)a.e.weights | (uintptr_t)a.e.positions |
                       (uintptr_t)a.e.weights_out | (uintptr_t)a.e.positions_out;
  if (a.e.cols % 4 == 0 && at % 16 == 0)
    k_evict_plan<THREADS, kVecs, FUSED, true><<<pairs, THREADS, 0, st>>>(a);
  else
    k_evict_plan<THREADS, kVecs, FUSED, false><<<pairs, THREADS, 0, st>>>(a);
}
template <bool FUSED>
void plan(const EvictArgs &a, hipStream_t st) {
  const unsigned pairs = (unsigned)(a.e.rows * a.e.heads);
  if (FUSED && a.e.cols <= 64)  // at most 128 moves
    k_evict_plan_small<64><<<pairs, 64, 0, st>>>(a);
  else if (FUSED && a.e.cols <= 256)
    k_evict_plan_small<256><<<pairs, 256, 0, st>>>(a);
  else if (a.e.cols <= 1024)
    launch_plan<256, 1, FUSED>(a, st);
  else if (a.e.cols <= 8192)
    launch_plan<512, 4, FUSED>(a, st);
  else if (a.e.cols <= 16384)
    launch_plan<1024, 4, FUSED>(a, st);
  else if (a.e.cols <= 32768)
    launch_plan<1024, 8, FUSED>(a, st);
  else if constexpr (!FUSED)
    k_evict_plan_long<1024><<<pairs, 1024, 0, st>>>(a);
  DGS_LAUNCH_CHECK();
}

// Few moves: the lists stay in LDS (rows of more than 32768 slots need them all the same).
bool few_moves(const EvictCall &e) { return evict_room(e) <= kFewMoves && e.cols <= 32768; }

}  // namespace

int64_t evict_workspace(const EvictCall &e) {
  const int64_t pairs = e.rows * e.heads;
  if (few_moves(e)) return 0;
  return up256(pairs * 4) + 2 * up256(pairs * evict_room(e) * 4);
}

void evict_rows(const EvictCall &e, void *ws, int64_t ws_bytes, hipStream_t st) {
  const int64_t pairs = e.rows * e.heads;
  if (pairs <= 0) return;
  const int64_t need = evict_workspace(e);
  DGS_CHECK(ws_bytes >= need && (need == 0 || ws), "evict: workspace too small");
  DGS_CHECK(pairs < (int64_t(1) << 31) && e.cols < (int64_t(1) << 30) &&
                e.page < (int64_t(1) << 31),
            "evict: too many rows or columns");
  EvictArgs a{};
  a.e = e;
  a.room = evict_room(e);
  a.gd = state_guard();
  if (few_moves(e)) {
    plan<true>(a, st);
    return;
  }
  char *w = static_cast<char *>(ws);
  a.moves = (int32_t *)w;
  a.holes = (int32_t *)(w + up256(pairs * 4));
  a.movers = (int32_t *)(w + up256(pairs * 4) + up256(pairs * a.room * 4));
  plan<false>(a, st);
  // no slot can go from rows that the budget covers (long ones come this way too)
  if (e.nstores == 0 || a.room == 0) return;
  // enough blocks to fill the card, at least 8 rows for each of a block's groups
  int64_t ny = ceil_div(a.room, 128);
  const int64_t fill = ceil_div(4096, pairs);
  if (ny > fill) ny = fill;
  if (ny > 1024) ny = 1024;
  const dim3 grid((unsigned)pairs, (unsigned)ny, (unsigned)e.nstores);
  k_evict_move<<<grid, kMoveThreads, 0, st>>>(a);
  DGS_LAUNCH_CHECK();
}

}  // namespace dgs
