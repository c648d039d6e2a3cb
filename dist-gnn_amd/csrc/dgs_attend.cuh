// dgs_attend.cuh -- what the kernels of the attention over the 4-bit state cache share, and its
// matrix form (state_attend.hip has the operator, its vector form and the joining of splits).
#pragma once

#include "dgs_lane.cuh"
#include "dgs_state.cuh"

namespace dgs {

struct AttendArgs {
  StateView c;
  const void *q;
  int64_t q_row, q_head;
  int64_t rows;
  int q_heads, g;  // g = query heads per head
  IdArray table, lens;
  int64_t width;
  float scale2;  // scale * log2 e, below 2^101
  // How the work is cut.  A "pair" is a row and up to `together` query heads of one head (matrix form
  // 16, vector form 4).  With `stream` waves, the pairs' tiles of 2^shift slots lie in a line that is
  // cut evenly over the waves; else the matrix form takes a workgroup a pair and the vector form
  // `splits` chunks of slots a row.  What is cut leaves parts: a (maximum, sum) and an unnormalised
  // output each.  Parts of a query head: with splits (row q_heads + head) splits + split, else
  // (pair + wave) * min(g, together) + query head, so that a pair's parts follow each other.
  int64_t chunk;
  int splits, stream, together;
  int shift, cost, least;  // of the line: see row_units, stream_share
  float *part_o;    // [parts, dim]
  float2 *part_ml;  // [parts]
  float *logits;   // [rows, q_heads, cap] (weights)
  int64_t cap;     // width << pshift
  float *weights;
  int64_t weights_cols;
  float decay;
  void *out;
  StateGuard gd;
};

// The matrix form for channel groups of 32, 64 or 128 and head_dim / group of 1, 2 or 4
// (state_m*.hip): workgroups of `waves` waves.
void attend_matrix_32(const AttendArgs &a, int waves, int type, hipStream_t st);
void attend_matrix_64(const AttendArgs &a, int waves, int type, hipStream_t st);
void attend_matrix_128(const AttendArgs &a, int waves, int type, hipStream_t st);
// Words of LDS that a wave of it needs.
inline int attend_matrix_lds(int dim, int group, int g, bool stream) {
  const int join = stream ? 0 : 32 + (g < 16 ? g : 16) * dim, corner = 8 * dim + 64 * (dim / group);
  return join > corner ? join : corner;
}
constexpr int kStreamRows = 1024;  // rows whose lengths a wave of the stream form adds up

namespace {

__device__ __forceinline__ int64_t row_length(const AttendArgs &a, int64_t row, bool report) {
  const int64_t len = a.lens[row];
  if ((uint64_t)len > (uint64_t)a.cap) {
    if (report) report_bad_id(a.gd.err, kAsyncErrLength, len, a.cap + 1, a.gd.tag);
    return len < 0 ? 0 : a.cap;
  }
  return len;
}

// A sum of probabilities is 0 where no slot is left, because every page lies outside the cache: the
// output is zeros then and the weights get nothing.  It is 0 too where every logit is -infinity, which
// has no softmax (NaN).  The maximum tells them apart: -infinity where no slot is left, kNoSoftmax,
// which every finite logit passes by far, where there is one.
constexpr float kNoSoftmax = -3.4028235e38f;
__device__ __forceinline__ float inverse_sum(float m, float l) { return m == -INFINITY ? 0.f : 1.f / l; }
// Whether one of the slots [first, last) of a row lies in the cache.  The lanes of a wave look together,
// or each for itself (kTogether = 1, rows of a few slots).
template <int kTogether>
__device__ __forceinline__ bool some_left(const AttendArgs &a, int64_t row, int first, int last) {
  const int end = (int)((last + (int64_t(1) << a.c.pshift) - 1) >> a.c.pshift);
#pragma unroll 1
  for (int p0 = first >> a.c.pshift; p0 < end; p0 += kTogether) {
    const int p = p0 + (kTogether > 1 ? (int)(threadIdx.x & 63) : 0);
    const bool in = p < end && (uint64_t)a.table[row * a.width + p] < (uint64_t)a.c.pages;
    if (kTogether > 1 ? __any(in) : in) return true;
  }
  return false;
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

// The stream form's line of units: rows in order, a row's pairs in order, and of a pair `cost` units
// for taking it up, then its tiles of 2^shift slots.
__device__ __forceinline__ int units_of(int len, int shift, int cost) {
  const int tiles = (int)(((int64_t)len + (1 << shift) - 1) >> shift);
  return tiles ? tiles + cost : 0;
}
__device__ __forceinline__ int row_units(const AttendArgs &a, int64_t row, int shift, int cost) {
  return units_of((int)row_length(a, row, false), shift, cost);
}
// Lane l adds up rows [l n / 64 ..): the line up to its rows, what its rows hold, the last one's length.
__device__ __forceinline__ void stream_sums(const AttendArgs &a, int shift, int cost, int lane,
                                            int per, int &before, int &own, int &total, int &len) {
  own = len = 0;
  for (int i = 0; i < per; ++i) {
    const int64_t r = (int64_t)lane * per + i;
    if (r < a.rows) {
      len = (int)row_length(a, r, false);
      own += units_of(len, shift, cost);
    }
  }
  int x = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  before = x - own;
  total = __builtin_amdgcn_readlane(x, 63);
}
// Units a wave takes: at least a pair's cost and `least` tiles.
__device__ __forceinline__ int stream_share(const AttendArgs &a, int cost, int least, int64_t units) {
  const int64_t q = (units + a.stream - 1) / a.stream;
  return (int)(q < least + cost ? least + cost : q);
}
// A wave's units [at, end) of the line, and where it is in them: a pair of a row, of which it takes
// the tiles from `tile` on and the slots before last().  All in scalar registers.
struct Run {
  int64_t at, end, row;
  int pairs, len, units, pair, unit0, tile;

  __device__ __forceinline__ bool start(const AttendArgs &a, int shift, int cost, int least,
                                        int pairs_of_row, int wave, int lane) {
    pairs = pairs_of_row;
    const int per = (int)((a.rows + 63) >> 6);
    int before, own, total, last_len;
    stream_sums(a, shift, cost, lane, per, before, own, total, last_len);
    const int share = stream_share(a, cost, least, (int64_t)total * pairs);
    at = (int64_t)wave * share;
    end = at + share < (int64_t)total * pairs ? at + share : (int64_t)total * pairs;
    if (at >= end) return false;
    // the lane, then the row, that holds unit `at`
    const int64_t t = at / pairs;  // rows' boundaries are multiples of `pairs` in the line
    const uint64_t has = __ballot(before <= t && t < (int64_t)before + own);
    const int who = __ffsll((unsigned long long)has) - 1;
    int front = __builtin_amdgcn_readlane(before, who);
    if (per == 1) {
      row = who;
      len = __builtin_amdgcn_readlane(last_len, who);
    } else {
      int64_t r = (int64_t)who * per;
      // bounded also where a caller changes the lengths under the kernel, as is the loop of next()
      for (int i = 1;; ++i, ++r) {
        len = (int)row_length(a, r, false);
        const int u = units_of(len, shift, cost);
        if (t < front + u || i >= per || r + 1 >= a.rows) break;
        front += u;
      }
      row = __builtin_amdgcn_readfirstlane((int)r);
      len = __builtin_amdgcn_readfirstlane(len);
      front = __builtin_amdgcn_readfirstlane(front);
    }
    units = units_of(len, shift, cost);
    if (units == 0) return false;
    const int64_t in_row = at - (int64_t)front * pairs;
    pair = __builtin_amdgcn_readfirstlane((int)(in_row / units));
    unit0 = __builtin_amdgcn_readfirstlane((int)(in_row % units));
    tile = unit0 < cost ? 0 : unit0 - cost;
    return true;
  }
  // The end of this wave's slots of its pair (none of them: not past the first).
  __device__ __forceinline__ int last(int shift, int cost) const {
    const int64_t stop = (unit0 + (end - at) - cost) * ((int64_t)1 << shift);
    return stop < 0 ? 0 : (stop < len ? (int)stop : len);
  }
  __device__ __forceinline__ bool next(const AttendArgs &a, int shift, int cost) {
    at += units - unit0;
    if (at >= end) return false;
    unit0 = tile = 0;
    if (++pair == pairs) {
      pair = 0;
      do {
        if (++row >= a.rows) return false;
        len = __builtin_amdgcn_readfirstlane((int)row_length(a, row, false));
        units = units_of(len, shift, cost);
      } while (units == 0);
    }
    return end - at > cost;  // else the next wave has its tiles
  }
};
// Matrix form: tiles of 32 slots, and 6 units for a pair (three loads that wait for each other, the
// query, the write of its part: as long as some tiles.  64 rows of 1 to 8192 slots with weights:
// 98 us without, 78 us at 2 units, 63 to 65 at 4, 6 and 8).
constexpr int kMatrixShift = 5, kMatrixCost = 6, kMatrixLeast = 4;

// Matrix form, for 16-bit queries.  One wave takes up to 16 query heads of a head (the columns left
// over are zeros) through 32 slots at a time, in v_mfma_f32_16x16x32_bf16 (operands: lane l holds
// row or column l & 15 and the eight k of quarter l >> 4; result: column l & 15, rows 4 (l >> 4) + i).
//
//  - A code c of K becomes the bfloat16 0x3f80 | c << 3 = (16 + c) / 16, exactly, with a shift and a
//    mask-or a pair.  V's become 0x4300 | c = 128 + c, which spares one shift in four; the offset's sums,
//    and their rounding, are 8 times as large, which K cannot have: the attention weights of 16-bit
//    queries would be off by 4e-7 instead of 6e-8 (V's go into a 16-bit output).
//  - x = K q / 16: rows are slots, columns query heads, k channels; one product chain per channel group,
//    r_g = sum q (16 + c) / 16.  Then x = sum_g s_g r_g + sum_g (b_g / 16 - s_g) Q_g with Q_g = sum q over
//    the group; the second sum is one more product whose slot operand is the stored (s, b) words
//    themselves and whose other operand holds -Q_g and Q_g / 16 in three bfloat16 terms (24 bits).  The
//    scale follows the sums, so that large queries only overflow where their sums do.
//  - The result leaves eight slots of a query head in a lane, of which only GR = 4, 8 or 16 columns
//    are query heads.  With fewer than 16, the other columns' lanes take over their share of the
//    slots (lane 4 b + h of a row of 16 takes slots 2 b and 2 b + 1 of head h), with one lane move
//    a value: at 4 query heads the softmax is a quarter of the work.
//  - out = V p: rows are channels (16 units of GROUP / 16 channels of one group), columns query
//    heads, k slots (which slot counts as which k is free, so the layout of x is the layout of p).
//    a_g = p s_g is rounded to two bfloat16 terms (17 bits: one term's 2^-9 would show in the
//    output), and the 128 sum a_g that the codes' offset adds is taken out with the same rounded
//    terms, through a product with a constant operand.  sum p b_g is summed in 32 bits and added at the
//    end: an output is off by up to 2^-17 of its group's largest value, which 16 bits hide except where
//    values cancel (32-bit queries take the vector form).  The pairs of slots that a register of V holds
//    are made with v_perm_b32.
//  - m only follows the maximum when a logit passes it by 8 (in base 2): p stays below 2^8, and
//    the rescaling is a rare branch.
//  - Rows come in 16 bytes a lane, two tiles ahead in registers, and pass through the wave's own
//    corner of LDS, from which every lane takes its words: narrow loads straight to their lanes (26
//    a tile) kept the wave waiting for 60 % of its time.  A row's 16-byte pieces are stored in an
//    order that depends on the row, so that the rows a read touches lie in different banks.
//  - P16: pages of at least 16 slots; a load's rows lie in one page, whose address stays in scalar
//    registers.
// STREAM = false: a workgroup a pair (row, head, 16 query heads), for rows that are short or many; its
// waves take 32 slots in turn and join through LDS in wave order.  STREAM: every wave takes an equal
// run of the tiles of all pairs, however long the rows are, and leaves its parts of a pair; the
// finishing kernel joins them.
// 8 rows of 8 heads of 128 channels, 100 to 131 thousand slots, 4 query heads a head (1024 MB): 192 us,
// 5.3 TB/s, as fast as rows come.  64 rows of 1 to 8192 slots with weights (210 MB): 50 us, 4.2 TB/s.
// One row of 700 slots: 12 us, a chain of loads (length, pages, rows) and the waves' joining.
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
// Nibbles y of a word's halves as bfloat16: of K 1 + c / 16, of V 128 + c.  `magic`, 0x3f803f80 or
// 0x43004300, comes in a vector register: one instruction takes one constant from a scalar register, so
// with both there the mask-or would be two.
__device__ __forceinline__ uint32_t code_pair_k(uint32_t x, int y, uint32_t magic) {
  return ((y == 0 ? x << 3 : x >> (4 * y - 3)) & 0x00780078u) | magic;
}
__device__ __forceinline__ uint32_t code_pair_v(uint32_t x, int y, uint32_t magic) {
  return ((x >> (4 * y)) & 0x000f000fu) | magic;
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
// Lanes of a row of 16: those of `banks` (bit b: lanes 4 b .. 4 b + 3) take x of the lane n below
// (shr) or above (shl), the others keep old.
template <int kN, int kBanks>
__device__ __forceinline__ float row_shr(float old, float x) {
  return __int_as_float(dpp_keep<0x110 + kN, kBanks>(__float_as_int(old), __float_as_int(x)));
}
template <int kN>
__device__ __forceinline__ uint32_t row_shl(uint32_t x) {
  return (uint32_t)dpp_keep<0x100 + kN>((int32_t)x, (int32_t)x);
}
// A result's two halves (slots 4 (l >> 4) + i and 16 more) -> this lane's GR / 2 slots of head l % GR.
template <int GR>
__device__ __forceinline__ void spread(const f32x4 (&r)[2], float (&x)[GR / 2]) {
  if constexpr (GR == 16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = r[i >> 2][i & 3];
  } else if constexpr (GR == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = row_shr<8, 0xC>(r[0][i], r[1][i]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float t = row_shr<4, 0x2>(r[0][i], r[0][2 + i]);
      t = row_shr<8, 0x4>(t, r[1][i]);
      x[i] = row_shr<12, 0x8>(t, r[1][2 + i]);
    }
  }
}
// The inverse for values packed in pairs: the operand of the columns that are query heads.
template <int GR>
__device__ __forceinline__ void collect(const uint32_t (&w)[GR / 4], Op &op) {
  if constexpr (GR == 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) op.u[i] = w[i];
  } else if constexpr (GR == 8) {
    op.u[0] = w[0];
    op.u[1] = w[1];
    op.u[2] = row_shl<8>(w[0]);
    op.u[3] = row_shl<8>(w[1]);
  } else {
    op.u[0] = w[0];
    op.u[1] = row_shl<4>(w[0]);
    op.u[2] = row_shl<8>(w[0]);
    op.u[3] = row_shl<12>(w[0]);
  }
}

template <int NG, int GROUP, int QT, int GR, bool P16, bool STREAM>
__global__ __launch_bounds__(NG * GROUP == 256 ? 256 : 512, NG * GROUP == 256 ? 1 : 2)
    void k_attend_matrix(AttendArgs a, int type, int tiles) {
  constexpr int kD = NG * GROUP, kC = kD / 32, kU = GROUP / 16, kGC = GROUP / 32, kV = GR / 2;
  extern __shared__ float s_mem[];
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, q4 = lane >> 4;
  const int pairs = a.c.heads * tiles;  // of a row
  const int gs = a.g < 16 ? a.g : 16;
  Run run;
  if constexpr (STREAM) {
    if (!run.start(a, kMatrixShift, kMatrixCost, kMatrixLeast, pairs,
                   (int)blockIdx.x * waves + wave, lane)) return;
  } else {
    run.row = blockIdx.x / (uint32_t)pairs;
    run.pair = (int)(blockIdx.x % (uint32_t)pairs);
  }
  // slots of a row fit 32 bits (checked on the host)
  int len = STREAM ? run.len
                   : __builtin_amdgcn_readfirstlane(
                         (int)row_length(a, run.row, run.pair == 0 && threadIdx.x == 0));
  int h = run.pair / tiles, rt = run.pair - h * tiles;
  int gn = a.g - rt * 16 < 16 ? a.g - rt * 16 : 16;  // query heads, at most GR
  int64_t qh0 = run.row * a.q_heads + h * a.g + rt * 16;
  // the slots [first, last) this wave takes, every step-th tile of 32
  const int step = STREAM ? 32 : waves * 32;
  int j1 = STREAM ? run.tile * 32 : wave * 32;
  int last = STREAM ? run.last(kMatrixShift, kMatrixCost) : len;
  // logits grow with x: a negative scale is taken into q, and so is 0 (masked slots are -inf)
  const float sign = a.scale2 < 0.f ? -1.f : (a.scale2 == 0.f ? 0.f : 1.f);
  const float scale2 = a.scale2 == 0.f ? 1.f : 16.f * fabsf(a.scale2);
  uint32_t magic_k = 0x3f803f80u, magic_v = 0x43004300u;
  asm volatile("" : "+v"(magic_k), "+v"(magic_v));

  const int ps = a.c.pshift, mask = (1 << ps) - 1;
  const int unit = n * (GROUP / 32);  // byte of this lane's unit of V in a group's codes
  const uint32_t sel = GROUP == 128 ? 0x05040100u
                       : GROUP == 64 ? ((unit & 2) ? 0x07060302u : 0x05040100u)
                                     : (0x0c000c00u | (uint32_t)(unit & 3) |
                                        ((uint32_t)(4 + (unit & 3)) << 16));
  const uint32_t pages = (uint32_t)a.c.pages;

  // A tile is kPR x 64 pieces of 16 bytes: those of K, then those of V, row by row.  kL loads of a
  // lane; load i of the first kL / 2 (kPR = 1: the lower half of the wave) belongs to K.  kRows rows
  // a load; a lane meets kIds different slots.
  constexpr int kPR = kD / 32, kL = kPR, kRows = 64 / kPR > 32 ? 32 : 64 / kPR;
  constexpr int kIds = 32 / kRows;
  static_assert(!P16 || kRows <= 16, "a load's rows lie in one page");
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
  // this lane's slots after spread(): slot(i) = 16 (i >> 2) + 4 q4 + (i & 3), i = i0 + v
  const int i0 = GR == 16 ? 0 : (n / GR) * kV;
  const uint32_t *my_w = s_w + (16 * (i0 >> 2) + 4 * q4 + (i0 & 3)) * NG;  // of K; V's: + 32 NG

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
  const char *tab;  // the row's

  // P16: the first slot of load i's rows, the same for all lanes; else this lane's
  auto slot_of = [&](int j0, int i) {
    const int j = j0 + i * kRows + (P16 ? 0 : lrow);
    return j < last ? j : (P16 ? (last - 1) & ~(kRows - 1) : last - 1);
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
      if (P16) {
        id[i] = __builtin_amdgcn_readfirstlane(id[i]);
        id_hi[i] = __builtin_amdgcn_readfirstlane(id_hi[i]);
      }
      const bool out = id[i] >= pages || (wide && id_hi[i] != 0);
      if (out)
        report_bad_id(a.gd.err, kAsyncErrSlot,
                      wide ? (int64_t)((uint64_t)id_hi[i] << 32 | id[i]) : (int64_t)(int32_t)id[i],
                      pages, a.gd.tag);
      page[i] = out ? 0u : id[i];
      t.bad[i] = P16 ? (out ? ~0ull : 0ull) : __ballot(out);
    }
    load_ids(j0 + step);
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      // the first row of the load (P16) or this lane's, in rows of the cache
      const int64_t r = (((int64_t)page[i] * a.c.heads + h) << ps) + (slot_of(j0, i) & mask);
      const uint32_t lr = P16 ? lrow : 0;
      if constexpr (kPR == 1) {
        t.c[0] = *(const su32x4 *)((lane < 32 ? a.c.kc : a.c.vc) + r * 16);
      } else {
        const uint32_t at = lr * (kD / 2) + 16 * lpiece;
        t.c[i] = *(const su32x4 *)(a.c.kc + r * (kD / 2) + at);
        t.c[kIds + i] = *(const su32x4 *)(a.c.vc + r * (kD / 2) + at);
      }
#pragma unroll
      for (int y = 0; y < kW; ++y) {
        // word e of the row's 2 NG (kPR = 1: the lower lanes fetch K's, the upper V's)
        const int e = kPR == 1 ? (lane < 32 ? y : NG + y) : lpiece + y * kPR;
        const uint32_t *wp = (e < NG ? a.c.ks : a.c.vs) + r * NG;
        t.w[i][y] = e < 2 * NG ? wp[lr * NG + (e < NG ? e : e - NG)] : 0u;
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
  Op qv[QT][kC], qm;
  f32x4 o[NG][kU], co[NG];
  float cb[NG], m, ms, l;  // m, ms: in base 2, of head n % GR
  Op ones;
#pragma unroll
  for (int i = 0; i < 4; ++i) ones.u[i] = 0x43004300u;  // 128, the offset of V's codes

  // word g of this lane's slot v
  auto word_at = [&](const uint32_t *w, int v, int g) {
    return w[(GR == 16 ? 16 * (v >> 2) + (v & 3) : v) * NG + g];
  };
  auto compute = [&](int j0, const uint64_t *bad) {
    float x[kV];
    {
      f32x4 s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        Op av;
#pragma unroll
        for (int g = 0; g < 4; ++g)
          av.u[g] = g < NG ? s_w[(16 * i + n) * NG + (g < NG ? g : 0)] : 0u;
        s[i] = mfma(av, qm, f32x4{0.f, 0.f, 0.f, 0.f});
      }
      spread<GR>(s, x);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4 r[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        r[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = g * kGC; c < (g + 1) * kGC; ++c) {
          const uint32_t w = *(const uint32_t *)(kp[c % kKP] + 256 * kPR * i + 64 * (c / 4));
          Op k;
#pragma unroll
          for (int y = 0; y < 4; ++y) k.u[y] = code_pair_k(w, y, magic_k);
          r[i] = mfma(k, qv[0][c], r[i]);
          if constexpr (QT == 2) r[i] = mfma(k, qv[1][c], r[i]);
        }
      }
      float rx[kV];
      spread<GR>(r, rx);
#pragma unroll
      for (int v = 0; v < kV; ++v)
        x[v] = __builtin_fmaf(scale_of(word_at(my_w, v, g)), rx[v], x[v]);
    }
    uint32_t vw[kV][NG];
#pragma unroll
    for (int v = 0; v < kV; ++v)
#pragma unroll
      for (int g = 0; g < NG; ++g) vw[v][g] = word_at(my_w + 32 * NG, v, g);
    bool some = false;
#pragma unroll
    for (int i = 0; i < kIds; ++i) some |= bad[i] != 0;
    if (j0 + 32 > last || some) {
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const int i = i0 + v, r = 16 * (i >> 2) + 4 * q4 + (i & 3);
        bool out = j0 + r >= last;
        if (some)
#pragma unroll
          for (int y = 0; y < kIds; ++y)
            out |= r / kRows == y && ((bad[y] >> ((r % kRows) * kPR)) & 1);
        if (out) {
          x[v] = -INFINITY;
#pragma unroll
          for (int g = 0; g < NG; ++g) vw[v][g] = 0;
        }
      }
    }
    if (a.logits && n % GR < gn) {
      float *lp = a.logits + (qh0 + n % GR) * a.cap + j0;
#pragma unroll
      for (int v = 0; v < kV; ++v) {
        const int i = i0 + v, r = 16 * (i >> 2) + 4 * q4 + (i & 3);
        if (j0 + r < last) lp[r] = x[v] * scale2;
      }
    }
    float top = x[0];
#pragma unroll
    for (int v = 1; v < kV; ++v) top = fmaxf(top, x[v]);
    top *= scale2;
    if (__any(top > m + 8.f)) {
      if constexpr (GR < 16) top = fmaxf(top, lane_xor32<8>(top));
      if constexpr (GR < 8) top = fmaxf(top, lane_xor32<4>(top));
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
    for (int v = 0; v < kV; ++v) {
      x[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[v], scale2, -ms));
      l += x[v];
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t vq[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        vq[i] = *(const uint32_t *)(vp[g % kVP] + 16 * kPR * (16 * (i >> 2) + (i & 3)) +
                                    64 * (g / kVP));
      uint32_t wh[kV / 2], wl[kV / 2];
#pragma unroll
      for (int v = 0; v < kV / 2; ++v) {
        const uint32_t w0 = vw[2 * v][g], w1 = vw[2 * v + 1][g];
        cb[g] = __builtin_fmaf(x[2 * v], base_of(w0), cb[g]);
        cb[g] = __builtin_fmaf(x[2 * v + 1], base_of(w1), cb[g]);
        const float a0 = x[2 * v] * scale_of(w0), a1 = x[2 * v + 1] * scale_of(w1);
        wh[v] = pack_bf16(a0, a1);
        wl[v] = pack_bf16(a0 - __uint_as_float(wh[v] << 16),
                          a1 - __uint_as_float(wh[v] & 0xffff0000u));
      }
      Op hi, lo;
      collect<GR>(wh, hi);
      collect<GR>(wl, lo);
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
        for (int i = 0; i < 4; ++i) v.u[i] = code_pair_v(pair[j >> 2][i], j & 3, magic_v);
        o[g][j] = mfma(v, hi, o[g][j]);
        o[g][j] = mfma(v, lo, o[g][j]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  };

  // Two tiles a turn, each staged from its own registers, which then take the tile after the next.
  // Tiles past the end load the last slot again and are masked whole: without conditions in the
  // loop the accumulators keep one set of registers.  kOdd: short rows leave before such a tile, where
  // that spills nothing (700 slots 12.0 us instead of 13.4, 320 rows of 14 to 17 slots 16.4 and 18.8;
  // cut rows, whose waves meet one such tile in many, 2 % slower).
  constexpr bool kOdd = !STREAM && NG <= 2 && QT * GR < 32;
  auto turn = [&](int j0, Rows &t) {
    stage(t);
    uint64_t bad[kIds];
#pragma unroll
    for (int i = 0; i < kIds; ++i) bad[i] = t.bad[i];
    load_rows(j0 + 2 * step, t);
    compute(j0, bad);
  };
  auto over_columns = [&](float x) {
    if constexpr (GR < 16) x += lane_xor32<8>(x);
    if constexpr (GR < 8) x += lane_xor32<4>(x);
    x += xor16(x);
    return x + xor32(x);
  };
#pragma unroll 1
  while (true) {
    // the first tiles, then the query: its loads and arithmetic run while the rows are on their way
    tab = (const char *)a.table.p + ((run.row * a.width) << (wide ? 3 : 2));
    if (j1 < last) {
      load_ids(j1);
      load_rows(j1, t0);
      load_rows(j1 + step, t1);
    }

    // q in bfloat16 terms, in the order in which code_pair_k() yields a word's channels: 0 4 1 5 2 6 3 7
    float qsum[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) qsum[g] = 0.f;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (n < gn)
        load_q(type, a.q, run.row * a.q_row + (h * a.g + rt * 16 + n) * a.q_head + 32 * c + 8 * q4, x);
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
    // quarter 0 holds the first bfloat16 terms of (-Q_g, Q_g / 16), 1 the second, 2 the third
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
        qm.u[g] = pack_bf16(-t, t * 0.0625f);
      }
    }

    m = -INFINITY;
    ms = l = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      co[g] = f32x4{0.f, 0.f, 0.f, 0.f};
      cb[g] = 0.f;
#pragma unroll
      for (int j = 0; j < kU; ++j) o[g][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (j1 < last) {
#pragma unroll 1
      for (int j0 = j1; j0 < last; j0 += 2 * step) {
        turn(j0, t0);
        if (kOdd && j0 + step >= last) break;
        turn(j0 + step, t1);
      }
    }
    if constexpr (!STREAM) {
      break;
    } else {
      if (j1 < last) {
        // this wave's part of the pair; a pair that it holds whole is finished here
        const bool whole = run.tile == 0 && last == len;
        l = over_columns(l);
        const int64_t part = (run.row * pairs + run.pair + blockIdx.x * waves + wave) * gs + n;
        if (__any(l == 0.f) && some_left<64>(a, run.row, j1, last)) m = l == 0.f ? kNoSoftmax : m;
        const float inv = whole ? inverse_sum(m, l) : 1.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float c = over_columns(cb[g]);
          if (n < gn) {
            const int ch = g * GROUP + 4 * q4 * kU;
#pragma unroll
            for (int e = 0; e < 4 * kU; e += 8) {
              float x[8];
#pragma unroll
              for (int y = 0; y < 8; ++y)
                x[y] = (o[g][(e + y) % kU][(e + y) / kU] - co[g][(e + y) / kU] + c) * inv;
              if (whole)
                store_out(type, a.out, (qh0 + n) * kD + ch + e, x);
              else
                store8<kStateF32>(a.part_o, part * kD + ch + e, x);
            }
          }
        }
        if (q4 == 0 && n < gn) a.part_ml[part] = make_float2(m, l);
      }
      if (!run.next(a, kMatrixShift, kMatrixCost)) return;
      len = run.len;
      h = run.pair / tiles;
      rt = run.pair - h * tiles;
      gn = a.g - rt * 16 < 16 ? a.g - rt * 16 : 16;
      qh0 = run.row * a.q_heads + h * a.g + rt * 16;
      j1 = 0;
      last = run.last(kMatrixShift, kMatrixCost);
    }
  }

  __syncthreads();  // the corners become the joining area:
  // [waves][16] maxima, [waves][16] sums, [waves][gn][kD] outputs
  l = over_columns(l);
  if (j1 < last && __any(l == 0.f) && some_left<64>(a, run.row, 0, len)) m = l == 0.f ? kNoSoftmax : m;
  float *s_m = s_mem, *s_l = s_mem + waves * 16, *s_o = s_mem + waves * 32;
  if (q4 == 0) s_m[wave * 16 + n] = m;
  __syncthreads();
  float all = -INFINITY;
  for (int w = 0; w < waves; ++w) all = fmaxf(all, s_m[w * 16 + n]);
  const float f = __builtin_amdgcn_exp2f(m - (all == -INFINITY ? 0.f : all));
  if (q4 == 0) s_l[wave * 16 + n] = l * f;
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float c = over_columns(cb[g]);
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
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, ls = 0.f, mm = -INFINITY;
    for (int w = 0; w < waves; ++w) {
      mm = fmaxf(mm, s_m[w * 16 + hd]);
      ls += s_l[w * 16 + hd];
      const float *src = s_o + (w * gn + hd) * kD + ch;
#pragma unroll
      for (int y = 0; y < 8; ++y) acc[y] += src[y];
    }
    const float inv = inverse_sum(mm, ls);
#pragma unroll
    for (int y = 0; y < 8; ++y) acc[y] *= inv;
    store_out(type, a.out, (qh0 + hd) * kD + ch, acc);
    if (a.part_ml && ch == 0) a.part_ml[(run.row * pairs + run.pair) * gs + hd] = make_float2(mm, ls);
  }
  if (!a.logits || a.part_ml) return;
  // The row and all its query heads are this workgroup's: it adds the weights from the logits
  // that it has just written (visible to it after the barriers above).
  float mh[GR], ih[GR];
#pragma unroll
  for (int g = 0; g < GR; ++g) {
    float mm = -INFINITY, ls = 0.f;
    if (g < gn)
      for (int w = 0; w < waves; ++w) {
        mm = fmaxf(mm, s_m[w * 16 + g]);
        ls += s_l[w * 16 + g];
      }
    mh[g] = g < gn ? (mm == -INFINITY ? 0.f : mm) : INFINITY;  // no head: exp2(-inf) * 0
    ih[g] = g < gn ? inverse_sum(mm, ls) : 0.f;
  }
  const float *lg = a.logits + qh0 * a.cap;
  float *wr = a.weights + (run.row * a.c.heads + h) * a.weights_cols;
  for (int j = threadIdx.x; j < len; j += blockDim.x) {
    float sum = 0.f;
#pragma unroll
    for (int g = 0; g < GR; ++g)
      sum += __builtin_amdgcn_exp2f(lg[(g < gn ? g : 0) * a.cap + j] - mh[g]) * ih[g];
    wr[j] = a.decay != 0.f ? sum + a.decay * wr[j] : sum;
  }
}

template <int NG, int GROUP, int QT, int GR, bool STREAM>
void launch_matrix_gr(const AttendArgs &a, int waves, int type, hipStream_t st) {
  const int tiles = (a.g + 15) / 16;
  const int64_t blocks = STREAM ? ceil_div(a.stream, waves) : a.rows * a.c.heads * tiles;
  DGS_CHECK(blocks < (int64_t(1) << 31), "attend: too many rows in one call");
  const size_t lds = (size_t)waves * attend_matrix_lds(NG * GROUP, GROUP, a.g, STREAM) * 4;
  const unsigned grid = (unsigned)blocks, threads = waves * 64;
  if constexpr (NG * GROUP >= 128) {
    if (a.c.pshift >= 4) {
      k_attend_matrix<NG, GROUP, QT, GR, true, STREAM><<<grid, threads, lds, st>>>(a, type, tiles);
      DGS_LAUNCH_CHECK();
      return;
    }
  }
  k_attend_matrix<NG, GROUP, QT, GR, false, STREAM><<<grid, threads, lds, st>>>(a, type, tiles);
  DGS_LAUNCH_CHECK();
}
template <int NG, int GROUP, int QT, int GR>
void launch_matrix_st(const AttendArgs &a, int waves, int type, hipStream_t st) {
  if (a.stream)
    launch_matrix_gr<NG, GROUP, QT, GR, true>(a, waves, type, st);
  else
    launch_matrix_gr<NG, GROUP, QT, GR, false>(a, waves, type, st);
}
template <int NG, int GROUP, int QT>
void launch_matrix_qt(const AttendArgs &a, int waves, int type, hipStream_t st) {
  if (a.g <= 4)
    launch_matrix_st<NG, GROUP, QT, 4>(a, waves, type, st);
  else if (a.g <= 8)
    launch_matrix_st<NG, GROUP, QT, 8>(a, waves, type, st);
  else
    launch_matrix_st<NG, GROUP, QT, 16>(a, waves, type, st);
}
template <int NG, int GROUP>
void launch_matrix(const AttendArgs &a, int waves, int type, hipStream_t st) {
  if (type == kStateBF16)
    launch_matrix_qt<NG, GROUP, 1>(a, waves, type, st);
  else
    launch_matrix_qt<NG, GROUP, 2>(a, waves, type, st);
}

}  // namespace
}  // namespace dgs
