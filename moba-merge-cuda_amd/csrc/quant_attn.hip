// Attention of one new token per row over an 8-bit paged cache (quant.h), split over
// the tokens and joined.
//
// For row r and head h of kv head kh, over the tokens t that the head attends (all of
// the first `length`, or those of the chunks it selected):
//   s_t = scale s^k_t (q . c^k_t),  o = sum_t exp(s_t - m) s^v_t c^v_t / z,
//   z = sum_t exp(s_t - m),  lse = m + log z
// Codes are exact in the 16-bit types, so q . c runs on the matrix units in q's type
// with fp32 sums.  The weight w_t = exp(s_t - m) s^v_t has the range of s^v and is
// split in two bf16 parts (w = hi + lo, off by 2^-17 of w), each multiplied by the
// codes: bf16 for its range, two parts for fp16's precision.  At 128 dims the second
// product costs 8 of 24 matrix instructions (fp8) or of 28 (int8), in a kernel that waits
// for memory.
//
// Bound by the reads of codes and scales.  Work is cut into units of 128 tokens of a
// (row, kv head, block of query heads); all units of the call, laid end to end, are
// dealt to the workgroups in equal runs, so that rows of unlike lengths load every CU
// alike.  A workgroup finds its run by a scan of the rows' lengths (on the device: a
// call reads nothing back).  Where an entry spans several workgroups each writes a
// partial (o, m, z), and a second launch joins them in order: nothing depends on
// timing.
//
// A wave works on 32 tokens at a time.  Their codes come from memory into LDS by loads
// that pass no register, in whole rows and with no barrier, as the tile is the wave's
// own: it reads the tile into registers, sends for the next one, and computes.
//   S^T = K Q^T (16x16x32): a lane supplies 8 dims of a token; what it then holds are
//         the scores of 4 + 4 tokens for one head;
//   O^T = V^T P^T: those 8 weights are a lane's share of P^T as they are, if V^T is
//         supplied with the same 8 tokens, which the transposed LDS read does.
// Calls at 64 rows of 256 to 32K tokens, 32 / 8 heads of 128 dims, int8 (831 MB): 139 to
// 141 us, 5.9 TB/s, where a plain read of such blocks and their scales takes 139; the first
// form with codes loaded to registers two steps ahead took 172 in this kernel alone.  One
// row of 128K tokens of 2 kv heads of 64 dims, fp8 (36 MB): 18.4 us; under the profiler
// this kernel takes 14.4 of it and the join 4.7.
#include <algorithm>

#include "quant.h"
#include "../../include/moba_hip.h"

using namespace moba;

namespace {

typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kUnit = 128;      // tokens of a unit: one step of each of the 4 waves
constexpr int kMaxWgs = 768;    // of a launch, at most
// Shares of a workgroup, at least.  Calls, us, at 2, 4, 6, 8: 256 rows of 64 to 4K tokens, one
// kv head 24.4, 23.3, 22.8, 25.0, two 37.0, 36.5, 36.2, 36.8; one row of 128K tokens of 64 dims
// 20.3, 18.7, 18.5, 20.0, of 96 dims 23.4, 20.9, 19.9, 19.8; 128 rows of up to 300 tokens 12.1,
// 13.9, 13.8, 13.7; 64 rows of up to 32K within 1%.
constexpr int kRun = 6;
// Units' worth of time that beginning and ending an entry takes (its length, slot, pages,
// query and sums wait for each other, about 4 us).  Calls, us, at 0, 1, 2, 3, 4: 256 rows of 64
// to 4K tokens, one kv head 31.1, 25.4, 22.8, 21.7, 23.5, two 50.3, 39.2, 36.2, 35.0, 37.3; 64
// rows of up to 32K 157, 145, 139, 139, 142; 32 such rows of 256 dims 94, 83, 77, 77, 77, of 192
// 61.5, 58.7, 59.3, 60.9, 60.3; 32 rows of 512 tokens 13.6, 16.9, 15.4, 16.1, 14.6; 56 short rows
// of 256 dims 70.2, 64.1, 63.9, 63.6, 64.8; one row of 64K 17.0, 18.2, 18.3, 18.3, 18.3.
constexpr int kBegin = 2;
constexpr int kManyParts = 8;   // of an entry, above which a workgroup joins one head
constexpr int kMaxSlots = 16;   // chunks that a head selects
constexpr int kMaxItems = 16 * kMaxSlots;  // of an entry
constexpr float kSlack = 6.0f;  // log2 by which scores may pass the running maximum

struct AttnArgs {
  QuantPool pool;
  const uint16_t* q;
  int Hq, G, HB, NHB;           // query heads per kv head; blocks of 16 in an entry (1, or 2 if dense); entries per kv head
  int per_row;                  // entries per row: Hkv * NHB
  FastDiv by_row, by_nhb;       // per_row, NHB
  const int *q_seq, *lengths;
  int length_add, max_length;
  const int* selected;          // null: dense
  int slots, chunk, max_items;
  FastDiv by_chunk, by_d4, by_pieces;
  int2* items;                  // [entries][max_items]: chunk, mask of heads
  int* tokens;                  // [entries] tokens of the items, end to end
  int scan_n, scan_mult;        // dense: rows, entries per row; else entries, 1
  uint32_t* start;              // [scan_n + 1] first share of each
  int4* many;                   // [workgroups / kManyParts] the entry in which that run begins (join_kernel)
  float scale_log2;
  float *part_o, *part_ml;      // [2 workgroups][16 HB heads][D], [..][2]
  uint16_t* out;
  float* lse;
};

MOBA_DEV int cut_length(const AttnArgs& a, int length) {
  const int64_t n = (int64_t)length + a.length_add;
  return (int)(n < 0 ? 0 : n < a.max_length ? n : a.max_length);
}
// Tokens that row r attends at most: none for a slot that does not exist.
MOBA_DEV int row_length(const AttnArgs& a, int r) {
  const int s = a.q_seq[r];
  if (s < 0 || s >= a.pool.B) return 0;
  return cut_length(a, a.lengths[r]);
}
MOBA_DEV int scan_tokens(const AttnArgs& a, int i) {
  return a.selected != nullptr ? a.tokens[i] : row_length(a, i);
}
// Workgroups for T shares: all of the launch's, where each then has kRun of them or
// more (a run that ends inside an entry writes its sums of 16 heads, as much as a quarter
// of a unit's codes), else fewer of them; up to one a CU for fewer shares than that.
MOBA_DEV uint32_t sharers(uint32_t launched, uint32_t T) {
  return min(launched, max((T + kRun - 1) / kRun, min(T, 256u)));
}
MOBA_DEV uint32_t units_of(int tokens) { return ((uint32_t)tokens + kUnit - 1) / kUnit; }
// What an entry counts for in the deal: its units, and what beginning and ending it costs.
MOBA_DEV uint32_t shares_of(int tokens) { return tokens > 0 ? units_of(tokens) + kBegin : 0; }

// Workgroup w of W has shares [first(w), first(w + 1)) of T >= W.
struct Deal {
  uint32_t q, r;
  MOBA_DEV Deal(uint32_t T, uint32_t W) : q(T / W), r(T % W) {}
  MOBA_DEV uint32_t first(uint32_t w) const { return q * w + min(w, r); }
  MOBA_DEV uint32_t owner(uint32_t x) const {
    const uint32_t big = r * (q + 1);
    return x < big ? x / (q + 1) : r + (x - big) / q;
  }
};

// ----------------------------------------------------- the chunks of an entry
// One wave per (row, kv head, block of heads): the distinct chunks that its heads
// selected, in order of first occurrence, with the mask of the heads that did; the
// chunk that the row's length ends in goes last, so that the entry's tokens are
// whole chunks and then what is left.  Chunks behind the length are dropped.
__global__ __launch_bounds__(64) void union_kernel(AttnArgs a) {
  __shared__ int chunk_s[kMaxItems], first_s[kMaxItems], rank_s[kMaxItems];
  __shared__ uint32_t mask_s[kMaxItems];
  const int e = blockIdx.x, lane = threadIdx.x;
  const int r = e / a.per_row, kh = (e % a.per_row) / a.NHB, blk = e % a.NHB;
  const int g0 = blk * 16, heads = min(16, a.G - g0), E = heads * a.slots;
  const int len = row_length(a, r);
  const int* sel = a.selected + ((int64_t)r * a.Hq + kh * a.G + g0) * a.slots;
  for (int x = lane; x < E; x += 64) {
    const int c = sel[x];
    chunk_s[x] = c >= 0 && (int64_t)c * a.chunk < len ? c : -1;
    mask_s[x] = 0;
  }
  __syncthreads();
  int n = 0;
  for (int x0 = 0; x0 < E; x0 += 64) {
    const int x = x0 + lane;
    int first = -1;
    if (x < E && chunk_s[x] >= 0) {
      first = 0;
      while (chunk_s[first] != chunk_s[x]) ++first;
    }
    const uint64_t m = __ballot(first == x && x < E);
    if (x < E) {
      first_s[x] = first;
      rank_s[x] = n + __popcll(m & ((1ull << lane) - 1));
    }
    n += __popcll(m);
  }
  __syncthreads();
  for (int x = lane; x < E; x += 64)
    if (first_s[x] >= 0) atomicOr(&mask_s[first_s[x]], 1u << (x / a.slots));
  __syncthreads();
  // the last chunk of the row changes places with the last of the list
  const int tail = len > 0 ? (len - 1) / a.chunk : -1;
  int at = -1;
  for (int x0 = 0; x0 < E; x0 += 64) {
    const int x = x0 + lane;
    const uint64_t m = __ballot(x < E && first_s[x] == x && chunk_s[x] == tail);
    if (m) at = rank_s[x0 + __ffsll((unsigned long long)m) - 1];
  }
  int2* out = a.items + (int64_t)e * a.max_items;
  for (int x = lane; x < E; x += 64) {
    if (first_s[x] != x) continue;
    int to = rank_s[x];
    if (at >= 0) to = to == at ? n - 1 : to == n - 1 ? at : to;
    out[to] = make_int2(chunk_s[x], (int)mask_s[x]);
  }
  if (lane == 0)  // distinct chunks of [0, len): no more than len tokens
    a.tokens[e] = (int)((int64_t)n * a.chunk - (at >= 0 ? (tail + 1ll) * a.chunk - len : 0));
}

// ------------------------------------------------------------------ attention
constexpr int kWaves = 4;  // of a workgroup
// NT: 16-dim tiles of a head that the registers hold.  Workgroups of a CU: what registers
// allow without spills.  Measured with one more or one less (kernel, us): 64 rows of up
// to 32K, 128 dims: 3 162, 2 141, 1 173; 32 rows of 256 dims: 2 107, 1 76; of 192: 2 54,
// 1 62; 8 rows of 32 heads of 64 dims: 3 30, 2 31.5.
template <int NT> constexpr int occupancy() { return NT <= 6 ? 3 : NT <= 12 ? 2 : 1; }

// Where a step's tokens are, before the pool's rows are known.
struct Look {
  int page;
  uint32_t at;    // place in the page; ~0: no token
  uint32_t mask;  // heads that attend it (chunks)
};

// 16 bytes a lane from memory to LDS, lane l's to lds + 16 l; read once.  Out of the
// compiler's sight, which would wait for it before every later read of LDS; `receive`
// waits where the bytes are read.  (One wait state between M0 and the load that uses it.)
MOBA_DEV void load_tile(const uint8_t* from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt"
               :: "s"(lds), "v"(from) : "memory", "m0");
}
// Four words at a 16-byte border.
template <typename T> MOBA_DEV T lds4(const void* p) {
  return *reinterpret_cast<const T*>(__builtin_assume_aligned(p, 16));
}
typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2_t lds_i32x2_t;
// ds_read_b64_tr_b8: in each 16 lanes, lane i gets byte i of 8 rows of 16 bytes when lane
// i' addresses row i' / 2, byte 8 (i' % 2).
MOBA_DEV i32x2_t read_tr8(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_t*)p);
}

// What a lane knows of a step: the scales of token l of its 64 and the heads that attend
// it; which of the tokens there are, and which of those all heads attend.
struct Step {
  float ks, vs;
  uint32_t mask;
  uint64_t live, all;
};

// The query of a lane's head in the dims that the lane multiplies: as it is, for keys that
// are turned into its type; or, for int8 keys, which go to the matrix unit as they are, as
// three 8-bit digits of a 24-bit integer q 2^k with max |q| 2^k in [2^21, 2^22): off by
// at most 2^-22 of the largest |q|, and exact for what lies less than 2^11 (fp16) or
// 2^14 (bf16) below it.  Turning 128 dims of 32 int8 keys takes a wave 96
// instructions; joining three integer sums of 8 scores takes 40.
// Where a few values are so much larger than the rest that the digits lose what the rest
// add to a score, the wave multiplies its queries as they are, with the keys turned: as
// soon as for one head the digits' errors come to more than 2^-20 of sum min(|q|, 2^14
// units), in which a large value counts as one of 2^14 units (2^-8 to 2^-7 of the largest).
// Values of a normal distribution are far from that: one in 10^3 (fp16) or 10^4 (bf16) has
// an error.  64 rows of up to 32K with such queries: 173 us instead of 140; a loop of their
// own for them took 192 dims from 59 to 70 (registers).
template <int FMT, int NT> constexpr bool digits() { return FMT == 0 && NT > 4; }
template <int DT, int NT, bool DIGITS> struct Query;
template <int DT, int NT> struct Query<DT, NT, false> {
  static constexpr int kSteps = (NT + 1) / 2, kBytes = 8;  // of 32 dims: 8 of a lane's token
  static constexpr int kRaw = kSteps;
  static MOBA_DEV int dim(int c, int g) { return 32 * c + 8 * g; }
  u16x8_t part[kSteps];
  MOBA_DEV void set(const u16x8_t (&raw)[kRaw]) {
    u16x8_t top = zero8();
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      part[c] = raw[c];
      top = __builtin_elementwise_max(top, raw[c] & (uint16_t)0x7fff);
    }
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) bits = max(bits, (uint32_t)top[e]);
    // A query that is not finite: its scores are NaN.  As it is, keys of one sign would make
    // all of them -inf, which is what a row has that attends nothing.
    const uint64_t bad = __ballot(bits >= (DT == 0 ? 0x7f80u : 0x7c00u));
    if (bad != 0) {  // the same for all four lanes of a head
      const uint32_t nan = (bad >> (threadIdx.x & 15)) & 0x0001000100010001ull ? 0x7fff7fffu : 0u;
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
        part[c] = __builtin_bit_cast(u16x8_t, __builtin_bit_cast(u32x4_t, part[c]) | nan);
    }
  }
  struct Codes {
    uint2 step[kSteps];
    MOBA_DEV void read(int c, const uint8_t* p) { step[c] = *reinterpret_cast<const uint2*>(p); }
  };
  // q . c of a token's codes
  template <int FMT> MOBA_DEV f32x4_t dot(const Codes& k) const {
    f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      uint32_t w[4];
      numbers4_16<FMT, DT>(k.step[c].x, w[0], w[1]);
      numbers4_16<FMT, DT>(k.step[c].y, w[2], w[3]);
      s = mfma16<DT>(__builtin_bit_cast(u16x8_t, (u32x4_t){w[0], w[1], w[2], w[3]}), part[c], s);
    }
    return s;
  }
};
template <int DT, int NT> struct Query<DT, NT, true> {
  static constexpr int kSteps = (NT + 3) / 4, kBytes = 16;  // of 64 dims: 16 of a lane's token
  i32x4_t digit[3][kSteps];  // lowest first
  float unit;                // 2^-k
  bool whole;                // the digits do for all heads of the wave
  static constexpr int kRaw = 2 * kSteps;
  static MOBA_DEV int dim(int c, int g) { return 64 * (c >> 1) + 16 * g + 8 * (c & 1); }
  MOBA_DEV void set(const u16x8_t (&raw)[kRaw]) {
    uint32_t bits = 0;
#pragma unroll
    for (int c = 0; c < kRaw; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) bits = max(bits, __float_as_uint(to_f32<DT>(raw[c][e])) & 0x7fffffffu);
    }
    bits = max(bits, (uint32_t)__shfl_xor((int)bits, 16, 64));
    bits = max(bits, (uint32_t)__shfl_xor((int)bits, 32, 64));
    // a query that is not finite: its scores are NaN
    const bool finite = bits < 0x7f800000u;
    const int e = max((int)(bits >> 23), 1 + 21);  // max |q| < 2^(e - 126); smallest: 2^-105
    const float fold = __uint_as_float((uint32_t)(finite ? min(127 + 126 + 22 - e, 254) : 127) << 23);
    unit = finite ? __uint_as_float((uint32_t)max(e - 22 + 1, 0) << 23) : __uint_as_float(0x7fc00000u);
    float lost = 0.0f;  // in units; NaN for a query that is not finite, as its scores
#pragma unroll
    for (int c = 0; c < kSteps; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t d[3] = {0, 0, 0};
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int i = 4 * w + b;
          const float x = to_f32<DT>(raw[2 * c + (i >> 3)][i & 7]) * fold, near = rintf(x);
          lost += fabsf(x - near);
          int v = (int)near;
#pragma unroll
          for (int y = 0; y < 3; ++y) {
            d[y] |= ((uint32_t)v & 255u) << (8 * b);
            v = (v + 128) >> 8;  // what the signed digit leaves
          }
        }
#pragma unroll
        for (int y = 0; y < 3; ++y) digit[y][c][w] = (int)d[y];
      }
    whole = true;
    if (__any(lost > 0.0f)) {
      float held = 0.0f;
#pragma unroll
      for (int c = 0; c < kRaw; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) held += fminf(fabsf(to_f32<DT>(raw[c][i]) * fold), 0x1p14f);
#pragma unroll
      for (int off = 16; off < 64; off <<= 1) {
        lost += __shfl_xor(lost, off, 64);
        held += __shfl_xor(held, off, 64);
      }
      whole = !__any(lost > 0x1p-20f * held);
    }
  }
  struct Codes {
    i32x4_t step[kSteps];
    MOBA_DEV void read(int c, const uint8_t* p) { step[c] = *reinterpret_cast<const i32x4_t*>(p); }
  };
  template <int FMT> MOBA_DEV f32x4_t dot(const Codes& k) const {
    i32x4_t s[3];
#pragma unroll
    for (int x = 2; x >= 0; --x) {
      // the highest two digits in one integer: 127 256 (65 256 + 128) < 2^31
#pragma unroll
      for (int i = 0; i < 4; ++i) s[x][i] = x == 1 ? s[2][i] << 8 : 0;
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
        s[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k.step[c], digit[x][c], s[x], 0, 0, 0);
    }
    f32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = fmaf((float)s[1][i], 256.0f, (float)s[0][i]) * unit;
    return r;
  }
  // q . c of two tiles without digits; row: the query in memory, null for no head.
  MOBA_DEV void dot_as_it_is(const Codes (&k)[2], const uint16_t* row, int D, int g, f32x4_t (&s)[2]) const {
    s[0] = s[1] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < kRaw; ++c) {
      const int d = dim(c, g);
      u16x8_t x = zero8();
      if (row != nullptr && d < D) x = ld8(row + d);
      asm volatile("" ::: "memory");  // one load's registers at a time
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        uint32_t w[4];
        numbers4_16<0, DT>((uint32_t)k[t].step[c >> 1][2 * (c & 1)], w[0], w[1]);
        numbers4_16<0, DT>((uint32_t)k[t].step[c >> 1][2 * (c & 1) + 1], w[2], w[3]);
        s[t] = mfma16<DT>(__builtin_bit_cast(u16x8_t, (u32x4_t){w[0], w[1], w[2], w[3]}), x, s[t]);
      }
    }
    const float nan = unit - unit;  // of a query that is not finite
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[t][i] += nan;
  }
};

template <int DT, int FMT, int NT>
__global__ __launch_bounds__(256, occupancy<NT>()) void attend_kernel(AttnArgs a) {
  constexpr int LD = 16 * NT + 4;  // floats of a joined row: neighbouring heads 4 banks apart
  // a wave's tile (keys, then values of 32 tokens) and, when it has been used, its sums
  constexpr int TILE = 2 * 32 * 16 * NT, SUMS = 16 * LD * 4;
  __shared__ __attribute__((aligned(16))) uint8_t tile_s[kWaves][TILE > SUMS ? TILE : SUMS];
  __shared__ float join_m[kWaves][16], join_l[kWaves][16];
  __shared__ uint32_t off_s[kWaves][64];
  __shared__ __attribute__((aligned(16))) uint32_t mask_s[kWaves][64];
  __shared__ __attribute__((aligned(16))) float ks_s[kWaves][64], vs_s[kWaves][64];
  __shared__ int2 items_s[kMaxItems];
  __shared__ uint32_t wave_sum[kWaves], found[2];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c16 = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool moba = a.selected != nullptr;

  // ---- the run of shares that is this workgroup's
  const uint32_t per = ((uint32_t)a.scan_n + 255) / 256, i0 = tid * per;
  const uint32_t i1 = min(i0 + per, (uint32_t)a.scan_n);
  uint32_t mine = 0;
  for (uint32_t i = i0; i < i1; ++i) mine += shares_of(scan_tokens(a, i)) * a.scan_mult;
  uint32_t incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t below = __shfl_up(incl, off, 64);
    if (lane >= off) incl += below;
  }
  if (lane == 63) wave_sum[w] = incl;
  __syncthreads();
  uint32_t base = 0, T = 0;
#pragma unroll
  for (int x = 0; x < kWaves; ++x) {
    base += x < w ? wave_sum[x] : 0u;
    T += wave_sum[x];
  }
  uint32_t excl = base + incl - mine;
  const uint32_t W = sharers(gridDim.x, T);
  if (blockIdx.x == 0) {  // for the second launch
    uint32_t s = excl;
    for (uint32_t i = i0; i < i1; ++i) {
      a.start[i] = s;
      s += shares_of(scan_tokens(a, i)) * a.scan_mult;
    }
    if (tid == 0) a.start[a.scan_n] = T;
  }
  const int wg = xcd_contiguous(blockIdx.x, (int)W);
  if (wg < 0) return;  // also every workgroup of a call without tokens
  const Deal deal(T, W);
  const uint32_t x0 = deal.first(wg);
  uint32_t left = deal.first(wg + 1) - x0;
  if (x0 >= excl && x0 < excl + mine) {  // one thread has it
    uint32_t rem = x0 - excl, i = i0;
    for (; i + 1 < i1; ++i) {
      const uint32_t n = shares_of(scan_tokens(a, i)) * a.scan_mult;
      if (rem < n) break;
      rem -= n;
    }
    found[0] = i;
    found[1] = rem;
  }
  __syncthreads();
  uint32_t si = __builtin_amdgcn_readfirstlane(found[0]), off = __builtin_amdgcn_readfirstlane(found[1]), in = 0;
  bool first_segment = true;
  // Of every kManyParts-th run, for the second launch: the entry in which the run begins, its
  // first workgroup, parts (0: this run has none of it) and the row of the first one's partial.
  auto tell = [&](int e, uint32_t from, uint32_t shares, bool part) __attribute__((always_inline)) {
    if (!first_segment || tid != 0 || wg % kManyParts != 0) return;
    const uint32_t begin = x0 - from, w0 = deal.owner(begin);
    const uint32_t n = part ? deal.owner(begin + shares - kBegin - 1) - w0 + 1 : 0;
    a.many[wg / kManyParts] = make_int4(e, (int)w0, (int)n, (int)(2 * w0 + (deal.first(w0) < begin ? 1 : 0)));
  };
  // what the scan entry after the present one is, asked for while that one is worked on
  struct Peek {
    int tokens, slot, length;
  };
  auto peek = [&](uint32_t i) __attribute__((always_inline)) {
    Peek p;
    i = min(i, (uint32_t)a.scan_n - 1);
    const int r = moba ? (int)div_by(i, a.by_row) : (int)i;
    p.slot = a.q_seq[r];
    p.length = a.lengths[r];
    p.tokens = moba ? a.tokens[i] : 0;
    return p;
  };
  Peek coming = peek(si);

  while (left > 0) {
    // ---- a segment: n of entry e's units from `off` on; e is the in-th of scan entry si
    const int slot_id = __builtin_amdgcn_readfirstlane(coming.slot);
    int len = __builtin_amdgcn_readfirstlane(coming.length);
    len = slot_id < 0 || slot_id >= a.pool.B ? 0 : cut_length(a, len);
    const int scan_len = moba ? __builtin_amdgcn_readfirstlane(coming.tokens) : len;
    const uint32_t shares = shares_of(scan_len), u = units_of(scan_len);
    if (shares == 0) {
      coming = peek(++si);
      continue;
    }
    if (off >= shares) {  // at the start only: the run begins in a later entry of the row
      in = off / shares;
      off -= in * shares;
    }
    const uint32_t taken = min(left, shares - off), n = min(off + taken, u) - min(off, u);
    const int e = (int)(si * a.scan_mult + in);
    const uint32_t from = off;
    left -= taken;
    off += taken;
    if (off == shares) {
      off = 0;
      if (++in == (uint32_t)a.scan_mult) {
        in = 0;
        coming = peek(++si);
      }
    }
    if (n == 0) {  // the rest of an entry's shares, without units
      tell(e, from, shares, false);
      first_segment = false;
      continue;
    }
    const int r = (int)div_by(e, a.by_row), of_row = e - r * a.per_row;
    const int kh = (int)div_by(of_row, a.by_nhb), blk = of_row - kh * a.NHB;
    const int head0 = kh * a.G + blk * 16 * a.HB;             // of the entry
    const int heads = min(16 * a.HB, a.G - blk * 16 * a.HB);
    const int v_lo = (int)from * kUnit, v_hi = min((int)(from + n) * kUnit, scan_len);
    const int hb = w & (a.HB - 1), streams = kWaves >> (a.HB - 1), stream = w >> (a.HB - 1);
    const int my_head = hb * 16 + c16;                         // in the entry
    // A wave's step is 64 tokens, found with one look; 32 where 64 would leave waves idle.
    const bool uneven = a.HB == 1 && (n & 1) && n <= 8;
    const int span_log = uneven || v_hi - v_lo <= 32 * streams ? 5 : 6;
    const int steps = (v_hi - v_lo + (1 << span_log) - 1) >> span_log;
    const int* trow = a.pool.table + (int64_t)slot_id * a.pool.W;
    if (moba) {
      const int first_item = (int)div_by(v_lo, a.by_chunk), last_item = (int)div_by(v_hi - 1, a.by_chunk);
      const int2* it = a.items + (int64_t)e * a.max_items;
      for (int x = first_item + tid; x <= last_item; x += 256) items_s[x] = it[x];
      __syncthreads();
    }

    typedef Query<DT, NT, digits<FMT, NT>()> Q;
    u16x8_t raw[Q::kRaw];  // asked for first: its address waits for nothing
    {
      const uint16_t* qp = a.q + ((int64_t)r * a.Hq + head0 + min(my_head, heads - 1)) * a.pool.D;
#pragma unroll
      for (int c = 0; c < Q::kRaw; ++c) {
        const int d = Q::dim(c, g);
        raw[c] = ld8(qp + (d < a.pool.D ? d : 0));
      }
    }
    f32x4_t acc[NT];  // dims 16 t + 4 g + i of the lane's head
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;

    const uint32_t heads_mask = moba ? (1u << heads) - 1 : 0;  // selected chunks: heads <= 16
    const int pieces = a.pool.Dp / 16;  // of a row of codes
    // Piece p of token t's row lies at place p ^ f(t) of its row in the tile, so that the
    // same piece of 16 tokens lies in as many banks as it can (rows of 2^n pieces; the
    // others' strides spread it by themselves).
    const int f_shift = pieces == 8 ? 1 : pieces == 4 ? 2 : pieces == 2 ? 3 : 0;
    const int f_mask = (pieces & (pieces - 1)) == 0 ? pieces - 1 : 0;
    uint8_t* const tile = tile_s[w];
    uint8_t* const tile_v = tile + 32 * 16 * NT;
    const uint32_t tile_at = lds_addr(tile);
    auto look = [&](int step) __attribute__((always_inline)) {
      Look x;
      const int v = v_lo + (step << span_log) + lane;
      uint32_t t = v;
      x.mask = heads_mask;
      bool ok = lane < (1 << span_log) && v < v_hi;
      if (moba) {
        const uint32_t it = div_by(ok ? v : v_lo, a.by_chunk);
        const int2 item = items_s[it];
        t = item.x * a.chunk + ((ok ? v : v_lo) - it * a.chunk);
        x.mask = item.y;
        ok = ok && t < (uint32_t)len;
      }
      t = ok ? t : 0u;
      const uint32_t lp = div_by(t, a.pool.by_page);
      x.page = trow[lp];
      x.at = ok ? t - lp * a.pool.by_page.d : ~0u;
      return x;
    };
    // Puts a step's places, from its page entries, where all lanes see them, and asks for
    // the scales of the lane's token.  A step behind the last, and a token that is not
    // there, reads the pool's first row: such loads are cheaper than a branch around
    // them, behind which the compiler would wait for every load in flight.
    auto place = [&](const Look& x, Step& s) __attribute__((always_inline)) {
      const bool ok = x.at != ~0u && (uint32_t)x.page < (uint32_t)a.pool.num_pages;
      const uint32_t row = ok ? ((uint32_t)x.page * a.pool.Hkv + kh) * a.pool.P + x.at : 0u;
      off_s[w][lane] = row * (uint32_t)pieces;
      s.live = __ballot(ok);
      s.mask = x.mask;
      s.all = moba ? s.live & __ballot(x.mask == heads_mask) : s.live;
      s.ks = a.pool.ks[row];
      s.vs = a.pool.vs[row];
      wave_lds_sync();
    };
    // Keys and values of the 32 tokens from `half` (0 or 32) on are sent for in whole rows:
    // lane l of load j has place x = 64 j + l of the tile, of token x / pieces.
    uint32_t places[NT / 2];  // token, and piece above it
#pragma unroll
    for (int j = 0; j < NT / 2; ++j) {
      const int x = 64 * j + lane, t = (int)div_by(x, a.by_pieces), p = x - t * pieces;
      places[j] = x < 32 * pieces ? t | (p ^ ((t >> f_shift) & f_mask)) << 16 : 31;  // else: behind the rows
    }
    uint32_t source[NT / 2];  // 16-byte piece of the pool for each place
    auto aim = [&](int half) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) source[j] = off_s[w][half + (places[j] & 63)] + (places[j] >> 16);
    };
    auto send = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NT / 2; ++j) {
        if (2 * j < pieces) {
          load_tile(a.pool.k + ((uint64_t)source[j] << 4), tile_at + 1024 * j);
          load_tile(a.pool.v + ((uint64_t)source[j] << 4), tile_at + 32 * 16 * NT + 1024 * j);
        }
      }
    };
    // The tile's keys and values, as the products take them.
    typename Q::Codes keys[2];  // of token 16 t + l % 16
    i32x2_t values[NT];         // dim 16 t + l % 16 of tokens 4 g + j and 16 + 4 g + j, j < 4
    // (addresses are put together where they are used: held, they cost a wave of a SIMD)
    const uint32_t key_at = c16 * a.pool.Dp + (Q::kBytes == 16 ? 0 : 8 * (g & 1));
    const uint32_t key_f = 16 * ((c16 >> f_shift) & f_mask);  // the same for token 16 + c16
    const int token_v = (c16 & 8 ? 16 : 0) + 4 * g + ((c16 >> 1) & 3);
    const uint32_t value_at = token_v * a.pool.Dp + 8 * (c16 & 1);
    const uint32_t value_f = 16 * ((token_v >> f_shift) & f_mask);
    auto receive = [&]() __attribute__((always_inline)) {
      wait_vmcnt<0>();
      asm volatile("" ::: "memory");
      const uint32_t at_key = opaque(key_at), at_value = opaque(value_at);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < Q::kSteps; ++c) {
          // pieces behind the row: the query is 0 there, and the codes must be finite
          const int piece = Q::kBytes == 16 ? 4 * c + g : 2 * c + (g >> 1);
          keys[t].read(c, tile + at_key + t * 16 * a.pool.Dp + ((piece < pieces ? 16 * piece : 0) ^ key_f));
        }
#pragma unroll
      for (int t = 0; t < NT; ++t) values[t] = read_tr8(tile_v + at_value + ((t < pieces ? 16 * t : 0) ^ value_f));
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the tile may be sent for again
      asm volatile("" ::: "memory");
    };
    // Scales of a step, from a lane per token to where all lanes see them.
    auto share = [&](const Step& s) __attribute__((always_inline)) {
      ks_s[w][lane] = s.ks * a.scale_log2;
      vs_s[w][lane] = s.vs;
      if (moba) mask_s[w][lane] = s.mask;
      wave_lds_sync();
    };
    // Scores of 32 tokens in log2.
    Q query;
    f32x4_t sc[2];
    auto scores = [&](int half) __attribute__((always_inline)) {
      bool done = false;
      if constexpr (digits<FMT, NT>()) {
        if (__builtin_expect(!query.whole, 0)) {
          const int h = (int)opaque((uint32_t)my_head);  // (no address is held between halves)
          const uint16_t* row = a.q + ((int64_t)r * a.Hq + head0 + h) * a.pool.D;
          query.dot_as_it_is(keys, h < heads ? row : nullptr, a.pool.D, (int)opaque((uint32_t)g), sc);
          done = true;
        }
      }
      if (!done) {
#pragma unroll
        for (int t = 0; t < 2; ++t) sc[t] = query.template dot<FMT>(keys[t]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4_t kk = lds4<f32x4_t>(&ks_s[w][half + 16 * t + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[t][i] *= kk[i];
      }
    };
    // The softmax of those scores and their product with the values.
    auto weigh = [&](int half, const Step& s) __attribute__((always_inline)) {
      const uint32_t live = (uint32_t)(s.live >> half);
      const bool whole = (uint32_t)(s.all >> half) == ~0u;
      f32x4_t vv[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) vv[t] = lds4<f32x4_t>(&vs_s[w][half + 16 * t + 4 * g]);
      float p[8], wt[8], top = -INFINITY;
      uint32_t on = 0xff;  // bit j: the lane's head attends its token j
      if (!whole) {
        on = ((live >> (4 * g)) & 15) | (((live >> (16 + 4 * g)) & 15) << 4);
        if (moba) {
          uint32_t takes = 0;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const u32x4_t mk = lds4<u32x4_t>(&mask_s[w][half + 16 * t + 4 * g]);
#pragma unroll
            for (int i = 0; i < 4; ++i) takes |= ((mk[i] >> my_head) & 1) << (4 * t + i);
          }
          on &= takes;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sc[j >> 2][j & 3] = (on >> j) & 1 ? sc[j >> 2][j & 3] : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = sc[j >> 2][j & 3];
        top = fmaxf(top, p[j]);
      }
      // the maximum moves when a score passes it by a margin (the first finite score
      // does): weights of up to 2^6 lose nothing in fp32 and bf16
      if (__any(top > m + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float to = fmaxf(m, top), shrink = m == -INFINITY ? 0.0f : fast_exp2(m - to);
        m = to;
        l *= shrink;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][i] *= shrink;
      }
      const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = fast_exp2(p[j] - ref);
        l += p[j];
        wt[j] = p[j] * vv[j >> 2][j & 3];
      }
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) wt[j] = (on >> j) & 1 ? wt[j] : 0.0f;  // a NaN scale that is not attended
      }
      u32x4_t hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        hi[j] = pack2<0>(wt[2 * j], wt[2 * j + 1]);
        float x, y;
        unpack2<0>(hi[j], x, y);
        lo[j] = pack2<0>(wt[2 * j] - x, wt[2 * j + 1] - y);
      }
      if (live != ~0u) {  // a token that is not there: its codes were never written, or may be a NaN's
        uint32_t there[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t bits = (live >> (16 * x + 4 * g)) & 15;  // to a byte each
          there[x] = ((bits & 1) | (bits & 2) << 7 | (bits & 4) << 14 | (bits & 8) << 21) * 255u;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) values[t][x] &= (int)there[x];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        uint32_t v[4];
        numbers4_16<FMT, 0>((uint32_t)values[t][0], v[0], v[1]);
        numbers4_16<FMT, 0>((uint32_t)values[t][1], v[2], v[3]);
        const u16x8_t vt = __builtin_bit_cast(u16x8_t, (u32x4_t){v[0], v[1], v[2], v[3]});
        acc[t] = mfma16<0>(vt, __builtin_bit_cast(u16x8_t, hi), acc[t]);
        acc[t] = mfma16<0>(vt, __builtin_bit_cast(u16x8_t, lo), acc[t]);
      }
    };

    if (stream < steps) {
      // The halves of the wave's steps, in order: one is worked on, the next one's codes are
      // on their way, and where the one after lies is known, so that it can be sent for as
      // soon as the tile has been read.  Page entries are asked for one step ahead of that.
      // Everything a wave waits for in memory it waits for at the tile.
      struct Half {
        Step s;
        int half;
        bool any;
      } at, sent, aimed;
      int k = stream;
      Look page = look(k);
      Step step;
      bool second = false;
      auto prepare = [&]() __attribute__((always_inline)) {
        aimed.any = second || k < steps;
        aimed.half = second ? 32 : 0;
        if (second) {
          second = false;
        } else if (aimed.any) {
          place(page, step);
          k += streams;
          page = look(k);
          second = (step.live >> 32) != 0;
        }
        aimed.s = step;
        if (aimed.any) aim(aimed.half);
      };
      prepare();
      send();
      sent = aimed;
#pragma unroll
      for (int c = 0; c < Q::kRaw; ++c)
        if (Q::dim(c, g) >= a.pool.D || my_head >= heads) raw[c] = zero8();
      query.set(raw);  // while the tile is on its way: the next `prepare` waits for it
      prepare();
      do {
        at = sent;
        wave_prio<1>();  // the reads of the next half go out ahead of other waves' arithmetic
        receive();
        if (aimed.any) send();
        wave_prio<0>();
        sent = aimed;
        prepare();
        if (at.half == 0) share(at.s);
        scores(at.half);
        weigh(at.half, at.s);
      } while (sent.any);
    }

    tell(e, from, shares, true);
    // ---- the four waves join; head h of block hb is in waves hb, hb + HB, ...
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) {
      join_m[w][c16] = m;
      join_l[w][c16] = l;
    }
    wave_lds_sync();
    float* const sums = reinterpret_cast<float*>(tile);  // no load into the tile is on its way
#pragma unroll
    for (int t = 0; t < NT; ++t) *reinterpret_cast<f32x4_t*>(sums + c16 * LD + 16 * t + 4 * g) = acc[t];
    __syncthreads();
    const bool entire = n == u;
    const int D = a.pool.D;
    const int64_t slot = ((int64_t)2 * wg + (first_segment ? 0 : 1)) * 16 * a.HB;
    for (int x = tid; x < heads * (D / 4); x += 256) {
      const int h = (int)div_by(x, a.by_d4), d = 4 * (x - h * (D / 4)), b = h >> 4;
      float top = -INFINITY, z = 0.0f;
      for (int y = b; y < kWaves; y += a.HB) top = fmaxf(top, join_m[y][h & 15]);
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
      for (int y = b; y < kWaves; y += a.HB) {
        const float my = join_m[y][h & 15];
        const float f = my == -INFINITY ? 0.0f : fast_exp2(my - top);
        z += join_l[y][h & 15] * f;
        const f32x4_t v = *reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(tile_s[y]) + (h & 15) * LD + d);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] += v[i] * f;
      }
      if (entire) {
        const int64_t row = (int64_t)r * a.Hq + head0 + h;
        const float f = z == 0.0f ? 0.0f : 1.0f / z;
        *reinterpret_cast<uint2*>(a.out + row * D + d) =
            make_uint2(pack2<DT>(o[0] * f, o[1] * f), pack2<DT>(o[2] * f, o[3] * f));
        if (d == 0) a.lse[row] = z == 0.0f ? -INFINITY : (top + __log2f(z)) * kLn2;
      } else {
        *reinterpret_cast<f32x4_t*>(a.part_o + (slot + h) * D + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * (slot + h)) = make_float2(top, z);
      }
    }
    __syncthreads();  // the buffers are the next segment's
    first_segment = false;
  }
}

// Joins the partials of the entries that span several workgroups of the first launch:
// o = sum 2^(m_j - m) o_j, z = sum 2^(m_j - m) z_j, in an order that is fixed.  The
// first workgroups have an entry each: a thread has 4 dims of a head and all its parts.
// Entries of more than kManyParts parts are left to the others, one for each head and
// every kManyParts-th run: the entry in which that run begins is theirs if it is the
// first such run behind the entry's own begin; B / cols parts at once, cols threads of 4
// dims each (a power of two).  A launch of 4 to 7 us that waits: for where the parts are,
// then for maxima, sums and the first of the partials together.
struct Parts {
  uint32_t w0, n;     // first workgroup, and how many (0: no units)
  int64_t slot0;      // row of that one's partial of head 0
  int hpe;
  // workgroup w0 + j's: its first segment's (j > 0: its run begins within the entry)
  MOBA_DEV int64_t slot(uint32_t j) const { return j == 0 ? slot0 : (int64_t)2 * (w0 + j) * hpe; }
};
MOBA_DEV Parts parts_of(const AttnArgs& a, int e, int wgs) {
  Parts p;
  p.hpe = 16 * a.HB;
  const int si = a.scan_mult == 1 ? e : (int)div_by(e, a.by_row), in = e - si * a.scan_mult;
  const uint32_t T = a.start[a.scan_n], s0 = a.start[si], all = a.start[si + 1] - s0;
  const uint32_t shares = a.scan_mult == 1 ? all : div_by(all, a.by_row);
  p.w0 = p.n = 0;
  p.slot0 = 0;
  if (shares == 0) return p;
  const Deal deal(T, sharers(wgs, T));
  const uint32_t from = s0 + in * shares;
  p.w0 = deal.owner(from);
  p.n = deal.owner(from + shares - kBegin - 1) - p.w0 + 1;
  p.slot0 = ((int64_t)2 * p.w0 + (deal.first(p.w0) < from ? 1 : 0)) * p.hpe;
  return p;
}
template <int DT>
MOBA_DEV void store_joined(const AttnArgs& a, int64_t row, int d, const f32x4_t& o, float top, float z) {
  const float f = z == 0.0f ? 0.0f : 1.0f / z;
  *reinterpret_cast<uint2*>(a.out + row * a.pool.D + d) =
      make_uint2(pack2<DT>(o[0] * f, o[1] * f), pack2<DT>(o[2] * f, o[3] * f));
  if (d == 0) a.lse[row] = z == 0.0f ? -INFINITY : (top + __log2f(z)) * kLn2;
}

// 4 dims of a head, of N parts at most; the loads behind the last part repeat it.
template <int DT, int N> MOBA_DEV void join_few(const AttnArgs& a, const Parts& p, int64_t row, int h, int d) {
  float2 ml[N];
  f32x4_t v[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int64_t at = p.slot(min((uint32_t)j, p.n - 1)) + h;
    ml[j] = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
    v[j] = *reinterpret_cast<const f32x4_t*>(a.part_o + at * a.pool.D + d);
  }
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, z = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) top = fmaxf(top, ml[j].x);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if ((uint32_t)j >= p.n) break;
    const float f = ml[j].x == -INFINITY ? 0.0f : fast_exp2(ml[j].x - top);
    z += f * ml[j].y;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += v[j][i] * f;
  }
  store_joined<DT>(a, row, d, o, top, z);
}

template <int DT, int B>
__global__ __launch_bounds__(B) void join_kernel(AttnArgs a, int wgs, int entries, int cols, int per_entry) {
  __shared__ float weight[kMaxWgs];
  __shared__ float red[2][B / 64];
  __shared__ __attribute__((aligned(16))) f32x4_t sums[B / 64][64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, D = a.pool.D;
  int e = blockIdx.x, h = 0;
  const bool many = e >= entries;
  Parts p;
  if (many) {
    const int run = ((e - entries) / per_entry + 1) * kManyParts;
    h = (e - entries) % per_entry;
    const int4 t = a.many[run / kManyParts];  // not written for a run that there is not
    if (run >= (int)sharers(wgs, a.start[a.scan_n])) return;
    e = t.x;
    p.w0 = (uint32_t)t.y;
    p.n = (uint32_t)t.z;
    p.hpe = 16 * a.HB;
    p.slot0 = (int64_t)t.w * p.hpe;
    if (p.n <= kManyParts || (p.w0 / kManyParts + 1) * kManyParts != (uint32_t)run) return;
  } else {
    p = parts_of(a, e, wgs);
    if (p.n == 1 || p.n > kManyParts) return;  // written by that workgroup; or left to the others
  }
  const int r = (int)div_by(e, a.by_row), of_row = e - r * a.per_row;
  const int kh = (int)div_by(of_row, a.by_nhb), blk = of_row - kh * a.NHB;
  const int heads = min(p.hpe, a.G - blk * p.hpe);
  const int64_t row0 = (int64_t)r * a.Hq + kh * a.G + blk * p.hpe;
  if (!many) {
    for (int x = tid; x < heads * (D / 4); x += B) {
      const int hx = (int)div_by(x, a.by_d4), d = 4 * (x - hx * (D / 4));
      if (p.n == 0) store_joined<DT>(a, row0 + hx, d, (f32x4_t){0.f, 0.f, 0.f, 0.f}, -INFINITY, 0.0f);
      else if (p.n <= 4) join_few<DT, 4>(a, p, row0 + hx, hx, d);
      else join_few<DT, kManyParts>(a, p, row0 + hx, hx, d);
    }
    return;
  }
  if (h >= heads) return;
  auto sums_of = [&](uint32_t j) { return *reinterpret_cast<const float2*>(a.part_ml + 2 * (p.slot(j) + h)); };
  const int c = tid & (cols - 1), d = 4 * c, groups = B / cols;
  const int at = d < D ? d : 0;  // columns behind D repeat the first
  auto part = [&](uint32_t j) { return *reinterpret_cast<const f32x4_t*>(a.part_o + (p.slot(j) + h) * D + at); };
  const uint32_t first = tid / cols;
  const float2 mine = sums_of(min((uint32_t)tid, p.n - 1));
  f32x4_t o = part(min(first, p.n - 1));
  float top = mine.x;
  for (uint32_t j = tid + B; j < p.n; j += B) top = fmaxf(top, sums_of(j).x);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if (lane == 0) red[0][w] = top;
  __syncthreads();
  for (int x = 0; x < B / 64; ++x) top = fmaxf(top, red[0][x]);
  float z = 0.0f;
  for (uint32_t j = tid; j < p.n; j += B) {
    const float2 ml = j == (uint32_t)tid ? mine : sums_of(j);
    const float f = ml.x == -INFINITY ? 0.0f : fast_exp2(ml.x - top);
    weight[j] = f;
    z += f * ml.y;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) z += __shfl_xor(z, off, 64);
  if (lane == 0) red[1][w] = z;
  __syncthreads();
  z = 0.0f;
  for (int x = 0; x < B / 64; ++x) z += red[1][x];
  const float f0 = weight[min(first, p.n - 1)];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = first < p.n ? o[i] * f0 : 0.0f;
#pragma unroll 4
  for (uint32_t j = first + groups; j < p.n; j += groups) {
    const f32x4_t x = part(j);
    const float f = weight[j];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += x[i] * f;
  }
  for (int off = cols; off < 64; off <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], off, 64);
  if (lane < cols) sums[w][lane] = o;
  __syncthreads();
  if (tid >= cols || d >= D) return;
  o = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  for (int x = 0; x < B / 64; ++x)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += sums[x][c][i];
  store_joined<DT>(a, row0 + h, d, o, top, z);
}

// Shape of a call: blocks of heads, entries, workgroups, and what its workspace holds.
struct Shape {
  int G, HB, NHB, max_items, wgs, join_threads;
  int64_t joins, entries, items_at, tokens_at, start_at, many_at, part_o_at, part_ml_at, bytes;
};
Shape shape_of(int Nq, int Hq, int Hkv, int D, int slots, int chunk, int max_length) {
  Shape s;
  s.G = Hq / Hkv;
  // Two blocks of heads in an entry read its codes once for both; one block an entry joins
  // half as wide sums and has twice as many entries.  32 heads of one kv head, 128 dims, us:
  // 32 rows of 100K tokens and more (950 MB) two 253, one 307; 64 rows of 20K (328 MB) 102 and
  // 115; of 6.7K (110 MB, which stays in the last-level cache) 47 and 46; of 1K 22.5 and 22.0.
  // The lengths are on the device: the rule goes by what max_length lets be read, so that
  // short rows in a long table pay a little (8 rows of 2K, 64 heads of 2, 15.5 instead of 14.2).
  // With selected chunks one block, always: each reads what its own 16 heads chose, where two
  // read the other's too.  64 rows of 100K, one and two: 4 chunks of 64 a head 35, 56; 4 of 512
  // 92, 128; 9 of 1024 of which heads share nine in ten 141, 189; that all heads agree on 64, 62.
  const int blocks = (s.G + 15) / 16;
  s.HB = slots == 0 && blocks % 2 == 0 && 2.0 * Nq * Hkv * max_length * code_width(D) > 256 << 20 ? 2 : 1;
  s.NHB = (s.G + 16 * s.HB - 1) / (16 * s.HB);
  s.entries = (int64_t)Nq * Hkv * s.NHB;
  s.max_items = std::min(s.G, 16) * slots;
  // as many workgroups as the card holds at once, but no more than there can be units
  const int per_cu = D > 192 ? 1 : D > 96 ? 2 : 3;  // occupancy()
  const int64_t longest = slots > 0 ? std::min<int64_t>((int64_t)s.max_items * chunk, max_length) : max_length;
  const int64_t units = s.entries * ((longest + kUnit - 1) / kUnit);
  s.wgs = (int)std::min<int64_t>(256 * per_cu, (units + 7) / 8 * 8);
  if (s.wgs < 8) s.wgs = 8;
  // Wide workgroups join entries of 128 parts and more, if the work is even (us, 512 and 1024
  // threads): 2 entries of 384 parts 6.2, 5.4; 64 entries of 8 parts of 32 heads 7.2, 12.2; 256
  // entries of 3 parts 4.9, 7.6.  (256 threads: 9.5, 10.0, 5.9.)
  s.join_threads = s.wgs >= 128 * s.entries ? 1024 : 512;
  s.joins = s.entries + (s.wgs - 1) / kManyParts * std::min(s.G, 16 * s.HB);  // workgroups
  auto take = [&](int64_t n) { const int64_t at = s.bytes; s.bytes += (n + 255) / 256 * 256; return at; };
  s.bytes = 0;
  s.items_at = take(slots > 0 ? s.entries * s.max_items * 8 : 0);
  s.tokens_at = take(slots > 0 ? s.entries * 4 : 0);
  s.start_at = take((std::max<int64_t>(slots > 0 ? s.entries : Nq, 1) + 1) * 4);
  s.many_at = take(((s.wgs - 1) / kManyParts + 1) * 16);
  const int64_t rows = 2ll * s.wgs * 16 * s.HB;
  s.part_o_at = take(rows * D * 4);
  s.part_ml_at = take(rows * 8);
  return s;
}

template <int DT, int FMT> void launch_attend(const AttnArgs& a, int wgs, hipStream_t st) {
  const dim3 grid(wgs), block(256);
  const int tiles = a.pool.Dp / 16;
  if (tiles <= 4) hipLaunchKernelGGL((attend_kernel<DT, FMT, 4>), grid, block, 0, st, a);
  else if (tiles <= 6) hipLaunchKernelGGL((attend_kernel<DT, FMT, 6>), grid, block, 0, st, a);
  else if (tiles <= 8) hipLaunchKernelGGL((attend_kernel<DT, FMT, 8>), grid, block, 0, st, a);
  else if (tiles <= 12) hipLaunchKernelGGL((attend_kernel<DT, FMT, 12>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((attend_kernel<DT, FMT, 16>), grid, block, 0, st, a);
}

template <int DT> void launch_join(const AttnArgs& a, const Shape& s, hipStream_t st) {
  int cols = 16;
  while (cols * 4 < a.pool.D) cols *= 2;
  const int entries = (int)s.entries, per_entry = std::min(a.G, 16 * a.HB);
  const dim3 grid((unsigned)s.joins), block(s.join_threads);
  if (s.join_threads == 1024) hipLaunchKernelGGL((join_kernel<DT, 1024>), grid, block, 0, st, a, s.wgs, entries, cols, per_entry);
  else hipLaunchKernelGGL((join_kernel<DT, 512>), grid, block, 0, st, a, s.wgs, entries, cols, per_entry);
}

// Tokens of a row, units and heads are counted in 31 bits, the threads of a launch in 32 (the
// runtime refuses a launch of more, by when the first one would have been made).
bool countable(const Shape& s, int max_length) {
  return max_length <= 0x7fff0000 && s.entries * ((max_length + kUnit - 1ll) / kUnit + kBegin) < 1ll << 31 &&
         s.entries * 16 * s.HB < 1ll << 31 && s.joins * s.join_threads < 1ll << 32;
}

}  // namespace

extern "C" int64_t moba_hip_quantized_attention_work(int Nq, int Hq, int Hkv, int D, int slots, int chunk,
                                                     int max_length) {
  if (Nq < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || (int64_t)Nq * Hq >= 1ll << 31 || D < 8 || D > 256 || slots < 0 ||
      slots > kMaxSlots || (slots > 0 && chunk < 1) || max_length < 1)
    return -1;
  const Shape s = shape_of(Nq, Hq, Hkv, D, slots, chunk, max_length);
  return countable(s, max_length) ? s.bytes : -1;
}

extern "C" int moba_hip_quantized_attention(const void* q, int dtype, int Nq, int Hq, int Hkv, int D,
                                            float scale, int format, const void* k_codes,
                                            const void* v_codes, const float* k_scale,
                                            const float* v_scale, int num_pages, int page_size,
                                            const int* table, int B, int table_width, const int* q_seq,
                                            const int* lengths, int length_add, int max_length,
                                            const int* selected, int slots, int chunk, void* work,
                                            void* out, float* lse, void* stream) {
  AttnArgs a;
  const int rc = quant_pool_of("quantized_attention", format, k_codes, v_codes, (float*)k_scale, (float*)v_scale,
                               num_pages, page_size, Hkv, D, table, B, table_width, a.pool);
  if (rc) return rc;
  if (dtype != 0 && dtype != 1) { moba_set_error("quantized_attention: dtype must be 0 (bf16) or 1 (fp16)"); return MOBA_ERR_ARG; }
  if (Nq < 1 || Hq < 1 || Hq % Hkv) { moba_set_error("quantized_attention: nonempty q, Hq a multiple of Hkv required"); return MOBA_ERR_ARG; }
  if (!(scale >= 0x1p-126f && scale <= 1e30f)) { moba_set_error("quantized_attention: scale must be in [2^-126, 1e30]"); return MOBA_ERR_ARG; }
  if (max_length < 1) { moba_set_error("quantized_attention: max_length must be positive"); return MOBA_ERR_ARG; }
  if ((selected != nullptr) != (slots > 0) || slots > kMaxSlots || (selected != nullptr && chunk < 1)) { moba_set_error("quantized_attention: selected chunks need 1 to 16 slots and a chunk size"); return MOBA_ERR_ARG; }
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)work) & 15) || work == nullptr) { moba_set_error("quantized_attention: q, out and work must be 16-byte aligned"); return MOBA_ERR_ARG; }
  if (max_length > (int64_t)table_width * page_size) { moba_set_error("quantized_attention: max_length exceeds what the table maps"); return MOBA_ERR_ARG; }
  chunk = std::min(chunk, max_length);  // a longer one ends where the row does
  const bool heads = (int64_t)Nq * Hq < 1ll << 31;
  const Shape s = heads ? shape_of(Nq, Hq, Hkv, D, slots, chunk, max_length) : Shape();
  if (!heads || !countable(s, max_length)) {
    moba_set_error("quantized_attention: more than 2^31 tokens of a row, units of 128 tokens or heads, or 2^32 threads of a launch");
    return MOBA_ERR_ARG;
  }
  char* p = (char*)work;
  a.q = (const uint16_t*)q;
  a.Hq = Hq; a.G = s.G; a.HB = s.HB; a.NHB = s.NHB; a.per_row = Hkv * s.NHB;
  a.by_row = fast_div(a.per_row); a.by_nhb = fast_div(s.NHB);
  a.q_seq = q_seq; a.lengths = lengths; a.length_add = length_add; a.max_length = max_length;
  a.selected = selected; a.slots = slots; a.chunk = chunk; a.max_items = s.max_items;
  a.by_chunk = fast_div(std::max(1, chunk)); a.by_d4 = fast_div(D / 4); a.by_pieces = fast_div(a.pool.Dp / 16);
  a.items = (int2*)(p + s.items_at); a.tokens = (int*)(p + s.tokens_at);
  a.scan_n = selected != nullptr ? (int)s.entries : Nq;
  a.scan_mult = selected != nullptr ? 1 : a.per_row;
  a.start = (uint32_t*)(p + s.start_at); a.many = (int4*)(p + s.many_at);
  a.scale_log2 = scale * kLog2e;
  a.part_o = (float*)(p + s.part_o_at); a.part_ml = (float*)(p + s.part_ml_at);
  a.out = (uint16_t*)out; a.lse = lse;
  hipStream_t st = (hipStream_t)stream;
  if (selected != nullptr) hipLaunchKernelGGL(union_kernel, dim3((unsigned)s.entries), dim3(64), 0, st, a);
  if (dtype == 0) { if (format == 0) launch_attend<0, 0>(a, s.wgs, st); else launch_attend<0, 1>(a, s.wgs, st); }
  else { if (format == 0) launch_attend<1, 0>(a, s.wgs, st); else launch_attend<1, 1>(a, s.wgs, st); }
  if (dtype == 0) launch_join<0>(a, s, st);
  else launch_join<1>(a, s, st);
  return moba_launch_status("quantized_attention");
}
