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
// The plan, one workgroup per (row, head): the budget-th best key by counting digits (keys are 32
// bits, larger is better, kept in LDS), then the slots in order, every wave a run of them: ties,
// holes and movers are numbered by counting lanes, so that three barriers join the waves.
// The moves are a kernel of their own, over all stores; where there can only be a few (a cache
// that takes single tokens) the plan's workgroup does them.
#include "dgs_block.cuh"
#include "dgs_state.cuh"

namespace dgs {
namespace {

constexpr int kMoveThreads = 256;
constexpr int kDigits = 2048;  // 11 bits: the sign, the exponent and two bits of the mantissa first
constexpr int kMaxKeys = 32768;  // keys that fit LDS (128 KB of 160)
constexpr int kFewMoves = 32;

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

// FUSED: this workgroup moves the rows too.
template <int THREADS, bool IN_LDS, bool FUSED>
__global__ __launch_bounds__(THREADS) void k_evict_plan(EvictArgs a) {
  constexpr int kWaves = THREADS / 64, kOwn = kDigits / THREADS;
  extern __shared__ uint32_t s_key[];
  __shared__ uint32_t s_hist[kDigits];
  __shared__ uint32_t s_scan[kWaves], s_cnt[3][kWaves];
  __shared__ int32_t s_max[kWaves];
  __shared__ uint32_t s_digit, s_left;
  const EvictCall &e = a.e;
  const int64_t pair = blockIdx.x;
  const int64_t row = pair / e.heads;
  const int h = (int)(pair % e.heads);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = evict_length(a, row, tid == 0 && h == 0), cols = (int)e.cols;
  const float *w = e.weights + pair * e.cols;
  const int32_t *pos = e.positions ? e.positions + pair * e.cols : nullptr;
  float *wo = e.weights_out + pair * e.cols;
  int32_t *po = e.positions_out + pair * e.cols;
  const int budget = (int)(e.budget < cols ? e.budget : cols);
  const int keep = n < budget ? n : budget;
  if (tid == 0) {
    if (h == 0) {
      if (e.lens.bytes == 8)
        ((int64_t *)e.lens_out)[row] = keep;
      else
        ((int32_t *)e.lens_out)[row] = keep;
    }
    if (n <= budget) a.moves[pair] = 0;
  }
  for (int j = keep + tid; j < cols; j += THREADS) {
    wo[j] = 0.f;
    po[j] = -1;
  }
  if (n <= budget) {
    for (int j = tid; j < n; j += THREADS) {
      wo[j] = w[j];
      po[j] = pos ? pos[j] : j;
    }
    return;
  }
  // the highest position + 1
  int32_t top = -1;
  if (pos) {
#pragma unroll 4
    for (int j = tid; j < n; j += THREADS) top = pos[j] > top ? pos[j] : top;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const int32_t x = __shfl_xor(top, o, 64);
      top = x > top ? x : top;
    }
    if (lane == 0) s_max[wave] = top;
    __syncthreads();
    for (int i = 0; i < kWaves; ++i) top = s_max[i] > top ? s_max[i] : top;
  } else {
    top = n - 1;
  }
  const int64_t newest = (int64_t)top + 1 - e.recent;
  auto fetch = [&](int j) {
    const int32_t p = pos ? pos[j] : j;
    return key_of(w[j], p < e.sinks || p >= newest);
  };
  auto key_at = [&](int j) { return IN_LDS ? s_key[j] : fetch(j); };
  // the keep-th largest key: digits of 11, 11 and 10 bits from the top
  uint32_t prefix = 0, left = (uint32_t)keep;
  int shift = 32;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    const uint32_t done = pass == 0 ? 0u : ~0u << shift;  // bits settled so far
    shift -= bits;
    for (int i = tid; i < kDigits; i += THREADS) s_hist[i] = 0;
    __syncthreads();
#pragma unroll 4
    for (int j = tid; j < n; j += THREADS) {
      uint32_t k;
      if (pass == 0) {
        k = fetch(j);
        if (IN_LDS) s_key[j] = k;
      } else {
        k = key_at(j);
      }
      if ((k & done) == prefix) atomicAdd(&s_hist[(k >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    // thread t owns kOwn digits counted from the largest: an ascending scan of them
    uint32_t mine[kOwn], sum = 0, total;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      mine[i] = s_hist[kDigits - 1 - (tid * kOwn + i)];
      sum += mine[i];
    }
    uint32_t before = block_exclusive_scan<THREADS>(sum, &total, s_scan);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (before < left && left <= before + mine[i]) {
        s_digit = kDigits - 1 - (tid * kOwn + i);
        s_left = left - before;
      }
      before += mine[i];
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
    __syncthreads();
  }
  // In slot order, wave by wave: of the slots whose key equals the threshold the first `left` stay.
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
  if (lane == 0) s_cnt[0][wave] = cnt;
  __syncthreads();
  const uint32_t tie0 = before_wave(s_cnt[0]);
  int32_t *holes = a.holes + pair * a.room, *movers = a.movers + pair * a.room;
  uint32_t nh = 0, nm = 0;
  for (int turn = 0; turn < 2; ++turn) {  // count, then write
    uint32_t ties = tie0;
    for (int b = j0; b < j1; b += 64) {
      const int j = b + lane;
      const bool in = j < j1;
      const uint32_t k = in ? key_at(j) : 0u;
      const bool tie = in && k == prefix;
      const uint64_t tb = __ballot(tie);
      const bool kept = in && (k > prefix || (tie && ties + __popcll(tb & below) < left));
      ties += __popcll(tb);
      const uint64_t hb = __ballot(in && !kept && j < budget);
      const uint64_t mb = __ballot(kept && j >= budget);
      if (turn == 1) {
        if ((hb >> lane) & 1) holes[nh + __popcll(hb & below)] = j;
        if ((mb >> lane) & 1) movers[nm + __popcll(mb & below)] = j;
        if (kept && j < budget) {
          wo[j] = w[j];
          po[j] = pos ? pos[j] : j;
        }
      }
      nh += __popcll(hb);
      nm += __popcll(mb);
    }
    if (turn == 0) {
      if (lane == 0) {
        s_cnt[1][wave] = nh;
        s_cnt[2][wave] = nm;
      }
      __syncthreads();
      nh = before_wave(s_cnt[1]);
      nm = before_wave(s_cnt[2]);
    }
  }
  uint32_t all = 0;
  for (int i = 0; i < kWaves; ++i) all += s_cnt[1][i];
  if (tid == 0) a.moves[pair] = (int32_t)all;
  __syncthreads();  // the lists are written (a workgroup's stores are visible to it past a barrier)
  for (uint32_t i = tid; i < all; i += THREADS) {
    const int32_t d = holes[i], s = movers[i];
    wo[d] = w[s];
    po[d] = pos ? pos[s] : s;
  }
  if constexpr (FUSED) {
    for (int st = 0; st < e.nstores; ++st)
      for (uint32_t i = wave; i < all; i += kWaves) {
        int64_t d[1] = {store_slot(a, row, h, holes[i])};
        int64_t s[1] = {store_slot(a, row, h, movers[i])};
        if (d[0] >= 0 && s[0] >= 0) move_store<1>(e.stores[st], s, d, lane, 6);
      }
  }
}

// Block (x, y, z): (row, head), a share of its moves, a store.  1 << lg lanes move a row (as many
// as it has 16-byte pieces, up to a wave), four rows at a time.
__global__ __launch_bounds__(kMoveThreads) void k_evict_move(EvictArgs a) {
  constexpr int kU = 4;
  const int64_t pair = blockIdx.x;
  const int64_t row = pair / a.e.heads;
  const int h = (int)(pair % a.e.heads);
  const int moves = a.moves[pair];
  const EvictStore &st = a.e.stores[blockIdx.z];
  int lg = 0;
  while (lg < 6 && (16 << lg) < st.row_bytes) ++lg;
  const int sub = threadIdx.x & ((1 << lg) - 1);
  const int groups = kMoveThreads >> lg, stride = groups * gridDim.y;
  const int32_t *holes = a.holes + pair * a.room, *movers = a.movers + pair * a.room;
  for (int i = blockIdx.y * groups + (threadIdx.x >> lg); i < moves; i += kU * stride) {
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

int64_t evict_room(const EvictCall &e) {
  const int64_t over = e.cols - e.budget;
  return over <= 0 ? 0 : (over < e.budget ? over : e.budget);
}
int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }

template <int THREADS, bool IN_LDS, bool FUSED>
void launch_plan(const EvictArgs &a, hipStream_t st) {
  const int64_t pairs = a.e.rows * a.e.heads;
  const size_t lds = IN_LDS ? (size_t)a.e.cols * 4 : 0;
  if (lds > 48 * 1024) {
    static const hipError_t once = hipFuncSetAttribute(
        (const void *)k_evict_plan<THREADS, IN_LDS, FUSED>,
        hipFuncAttributeMaxDynamicSharedMemorySize, kMaxKeys * 4);
    DGS_HIP(once);
  }
  k_evict_plan<THREADS, IN_LDS, FUSED><<<(unsigned)pairs, THREADS, lds, st>>>(a);
  DGS_LAUNCH_CHECK();
}
template <bool FUSED>
void plan(const EvictArgs &a, hipStream_t st) {
  if (a.e.cols <= 8192)
    launch_plan<256, true, FUSED>(a, st);
  else if (a.e.cols <= kMaxKeys)
    launch_plan<1024, true, FUSED>(a, st);
  else
    launch_plan<1024, false, FUSED>(a, st);
}

}  // namespace

int64_t evict_workspace(const EvictCall &e) {
  const int64_t pairs = e.rows * e.heads;
  return up256(pairs * 4) + 2 * up256(pairs * evict_room(e) * 4);
}

void evict_rows(const EvictCall &e, void *ws, int64_t ws_bytes, hipStream_t st) {
  const int64_t pairs = e.rows * e.heads;
  if (pairs <= 0) return;
  DGS_CHECK(ws && ws_bytes >= evict_workspace(e), "evict: workspace too small");
  DGS_CHECK(pairs < (int64_t(1) << 31) && e.cols < (int64_t(1) << 30) &&
                e.page < (int64_t(1) << 31),
            "evict: too many rows or columns");
  EvictArgs a{};
  a.e = e;
  a.room = evict_room(e);
  char *w = static_cast<char *>(ws);
  a.moves = (int32_t *)w;
  a.holes = (int32_t *)(w + up256(pairs * 4));
  a.movers = (int32_t *)(w + up256(pairs * 4) + up256(pairs * a.room * 4));
  a.gd = state_guard(kAsyncErrSlot, e.pages);
  if (a.room <= kFewMoves) {
    plan<true>(a, st);
    return;
  }
  plan<false>(a, st);
  if (e.nstores == 0) return;
  // enough blocks to fill the card, at least 8 rows for each of a block's groups
  int64_t ny = ceil_div(a.room, 128);
  const int64_t fill = ceil_div(4096, pairs);
  if (ny > fill) ny = fill;
  if (ny > 1024) ny = 1024;
  k_evict_move<<<dim3((unsigned)pairs, (unsigned)ny, (unsigned)e.nstores), kMoveThreads, 0, st>>>(a);
  DGS_LAUNCH_CHECK();
}

}  // namespace dgs
