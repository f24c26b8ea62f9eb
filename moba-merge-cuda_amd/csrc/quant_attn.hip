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
// codes: bf16 for its range, two parts for fp16's precision.  The second product costs
// 8 of 24 matrix instructions, in a kernel that waits for memory.
//
// Bound by the reads of codes and scales.  Work is cut into units of 128 tokens of a
// (row, kv head, block of query heads); all units of the call, laid end to end, are
// dealt to the workgroups in equal runs, so that rows of unlike lengths load every CU
// alike.  A workgroup finds its run by a scan of the rows' lengths (on the device: a
// call reads nothing back).  Where an entry spans several workgroups each writes a
// partial (o, m, z), and a second launch joins them in order: nothing depends on
// timing.
//
// A wave takes 32 tokens a step, straight from memory into registers:
//   S^T = K Q^T (16x16x32): a lane supplies 16 dims of a token at a time; what it then
//         holds are the scores of 4 + 4 tokens for one head;
//   O^T = V^T P^T: those 8 weights are a lane's share of P^T as they are, if V^T is
//         supplied with the same 8 tokens, which a lane loads for 4 NC neighbouring
//         dims each and turns into operands by byte permutations.
// No LDS tile and no barrier in the loop; LDS holds where the step's tokens are.
#include <algorithm>

#include "quant.h"
#include "../../include/moba_hip.h"

using namespace moba;

namespace {

constexpr int kUnit = 128;      // tokens of a unit: one step of each of the 4 waves
constexpr int kMaxWgs = 1024;   // of a launch, at most
constexpr int kMaxSlots = 16;   // chunks that a head selects
constexpr int kMaxItems = 32 * kMaxSlots;
constexpr float kSlack = 6.0f;  // log2 by which scores may pass the running maximum

struct AttnArgs {
  QuantPool pool;
  const uint16_t* q;
  int Hq, G, HB, NHB;           // query heads per kv head; blocks of 16 in an entry (1, 2); entries per kv head
  int per_row;                  // entries per row: Hkv * NHB
  const int *q_seq, *lengths;
  int length_add, max_length;
  const int* selected;          // null: dense
  int slots, chunk, max_items;
  FastDiv by_chunk, by_d4;
  int2* items;                  // [entries][max_items]: chunk, mask of heads
  int* tokens;                  // [entries] tokens of the items, end to end
  int scan_n, scan_mult;        // dense: rows, entries per row; else entries, 1
  uint32_t* start;              // [scan_n + 1] first unit of each
  float scale_log2;
  float *part_o, *part_ml;      // [2 workgroups][16 HB heads][D], [..][2]
  uint16_t* out;
  float* lse;
};

// Tokens that row r attends at most: none for a slot that does not exist.
MOBA_DEV int row_length(const AttnArgs& a, int r) {
  const int s = a.q_seq[r];
  if (s < 0 || s >= a.pool.B) return 0;
  const int64_t n = (int64_t)a.lengths[r] + a.length_add;
  return (int)(n < 0 ? 0 : n < a.max_length ? n : a.max_length);
}
MOBA_DEV int scan_tokens(const AttnArgs& a, int i) {
  return a.selected != nullptr ? a.tokens[i] : row_length(a, i);
}
MOBA_DEV uint32_t units_of(int tokens) { return ((uint32_t)tokens + kUnit - 1) / kUnit; }

// Workgroup w of W has units [first(w), first(w + 1)) of T >= W.
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
  const int g0 = blk * 16 * a.HB, heads = min(16 * a.HB, a.G - g0), E = heads * a.slots;
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
// Bytes of 4 tokens, dword by dword, to the bytes of each place: out[b] holds byte b
// of a, b, c and d.
MOBA_DEV void transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&out)[4]) {
  const uint32_t ab0 = __builtin_amdgcn_perm(b, a, 0x05010400), ab2 = __builtin_amdgcn_perm(b, a, 0x07030602);
  const uint32_t cd0 = __builtin_amdgcn_perm(d, c, 0x05010400), cd2 = __builtin_amdgcn_perm(d, c, 0x07030602);
  out[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100);
  out[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302);
  out[2] = __builtin_amdgcn_perm(cd2, ab2, 0x05040100);
  out[3] = __builtin_amdgcn_perm(cd2, ab2, 0x07060302);
}

// A read of bytes that this call reads once.
template <typename T> MOBA_DEV T load_once(const T* p) { return __builtin_nontemporal_load(p); }

// Keys of a step: 16 dims at 64 c + 16 g of token 16 t + l % 16.
template <int NC> struct Keys {
  u32x4_t reg[2][NC];
};
// Values of a step: the lane's 4 NC dims of tokens 4 g + j (j < 4) and 16 + 4 g + j - 4.
template <int NC> struct Values {
  uint32_t reg[8][NC];
  MOBA_DEV void load(int j, const uint8_t* p) {
    if constexpr (NC == 1) {
      reg[j][0] = load_once(reinterpret_cast<const uint32_t*>(p));
    } else {
      typedef uint32_t words __attribute__((ext_vector_type(NC)));
      const words x = load_once(reinterpret_cast<const words*>(p));
#pragma unroll
      for (int d = 0; d < NC; ++d) reg[j][d] = x[d];
    }
  }
  // The 8 tokens of each of the four dims of dword d, in bf16.
  template <int FMT> MOBA_DEV void operands(int d, u32x4_t (&out)[4]) const {
    if constexpr (FMT == 1) {  // 16 permutations, then two codes an instruction
      uint32_t x[4], y[4];
      transpose4(reg[0][d], reg[1][d], reg[2][d], reg[3][d], x);
      transpose4(reg[4][d], reg[5][d], reg[6][d], reg[7][d], y);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t lo, hi;
        numbers4_16<1, 0>(x[b], lo, hi); out[b][0] = lo; out[b][1] = hi;
        numbers4_16<1, 0>(y[b], lo, hi); out[b][2] = lo; out[b][3] = hi;
      }
    } else {  // int8: a conversion takes any byte of a word, and the halves are put together
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lo = (float)(int8_t)(reg[2 * j][d] >> (8 * b)), hi = (float)(int8_t)(reg[2 * j + 1][d] >> (8 * b));
          out[b][j] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302);
        }
    }
  }
};
// What a lane knows of a step: the scales of token l % 32 and the heads that attend it;
// which of the step's tokens there are, and whether all heads attend all 32.
struct Step {
  float ks, vs;
  uint32_t mask, live;
  bool whole;
};

// Waves of a workgroup.
constexpr int kWaves = 4;
// Workgroups of a CU that the registers allow.
template <int NC> constexpr int occupancy() { return NC == 1 ? 3 : 2; }

// Where a step's tokens are, before the pool's rows are known.
struct Look {
  int page;
  uint32_t at;    // place in the page; ~0: no token
  uint32_t mask;  // heads that attend it (chunks)
};

template <int DT, int FMT, int NC>
__global__ __launch_bounds__(256, occupancy<NC>()) void attend_kernel(AttnArgs a) {
  constexpr int LD = 64 * NC + 4;  // floats of a joined row: neighbouring heads 4 banks apart
  __shared__ __attribute__((aligned(16))) float join_o[kWaves][16][LD];
  __shared__ float join_m[kWaves][16], join_l[kWaves][16];
  __shared__ __attribute__((aligned(16))) uint32_t off_s[kWaves][32], mask_s[kWaves][32];
  __shared__ __attribute__((aligned(16))) float ks_s[kWaves][32], vs_s[kWaves][32];
  __shared__ int2 items_s[kMaxItems];
  __shared__ uint32_t wave_sum[kWaves], found[2];

  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c16 = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool moba = a.selected != nullptr;

  // ---- the run of units that is this workgroup's
  const uint32_t per = ((uint32_t)a.scan_n + 255) / 256, i0 = tid * per;
  const uint32_t i1 = min(i0 + per, (uint32_t)a.scan_n);
  uint32_t mine = 0;
  for (uint32_t i = i0; i < i1; ++i) mine += units_of(scan_tokens(a, i)) * a.scan_mult;
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
  const uint32_t W = min((uint32_t)gridDim.x, T);
  if (blockIdx.x == 0) {  // for the second launch
    uint32_t s = excl;
    for (uint32_t i = i0; i < i1; ++i) {
      a.start[i] = s;
      s += units_of(scan_tokens(a, i)) * a.scan_mult;
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
    for (;; ++i) {
      const uint32_t n = units_of(scan_tokens(a, i)) * a.scan_mult;
      if (rem < n) break;
      rem -= n;
    }
    found[0] = i;
    found[1] = rem;
  }
  __syncthreads();
  uint32_t si = __builtin_amdgcn_readfirstlane(found[0]), rem = __builtin_amdgcn_readfirstlane(found[1]);
  bool first_segment = true;

  while (left > 0) {
    // ---- a segment: units [off, off + n) of entry e
    const int scan_len = __builtin_amdgcn_readfirstlane(scan_tokens(a, si));
    const uint32_t u = units_of(scan_len);
    if (u == 0) { ++si; continue; }
    const uint32_t in = rem / u, off = rem - in * u, n = min(left, u - off);
    const int e = (int)(si * a.scan_mult + in);
    const int r = e / a.per_row, kh = (e % a.per_row) / a.NHB, blk = e % a.NHB;
    const int head0 = kh * a.G + blk * 16 * a.HB;             // of the entry
    const int heads = min(16 * a.HB, a.G - blk * 16 * a.HB);
    const int len = moba ? __builtin_amdgcn_readfirstlane(row_length(a, r)) : scan_len;
    const int v_lo = (int)off * kUnit, v_hi = min((int)(off + n) * kUnit, scan_len);
    const int hb = w % a.HB, streams = kWaves / a.HB, stream = w / a.HB;
    const int my_head = hb * 16 + c16;                         // in the entry
    const int steps = (v_hi - v_lo + 31) / 32;
    const int* trow = a.pool.table + (int64_t)a.q_seq[r] * a.pool.W;
    if (moba) {
      const int first_item = (int)div_by(v_lo, a.by_chunk), last_item = (int)div_by(v_hi - 1, a.by_chunk);
      const int2* it = a.items + (int64_t)e * a.max_items;
      for (int x = first_item + tid; x <= last_item; x += 256) items_s[x] = it[x];
      __syncthreads();
    }

    u16x8_t qf[2 * NC];  // dims 64 c + 16 g + 8 x .. + 7 of the lane's head
    {
      const uint16_t* qp = a.q + ((int64_t)r * a.Hq + head0 + min(my_head, heads - 1)) * a.pool.D;
#pragma unroll
      for (int c = 0; c < 2 * NC; ++c) {
        const int d = 64 * (c >> 1) + 16 * g + 8 * (c & 1);
        const u16x8_t x = ld8(qp + (d < a.pool.D ? d : 0));
        qf[c] = d < a.pool.D && my_head < heads ? x : zero8();
      }
    }
    f32x4_t acc[4 * NC];
#pragma unroll
    for (int t = 0; t < 4 * NC; ++t) acc[t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.0f;

    const uint32_t heads_mask = heads == 32 ? ~0u : (1u << heads) - 1;
    const uint32_t pieces = a.pool.Dp / 16;  // of a row of codes
    auto look = [&](int step) __attribute__((always_inline)) {
      Look x;
      const int v = v_lo + 32 * step + (lane & 31);
      uint32_t t = v;
      x.mask = heads_mask;
      bool ok = v < v_hi;
      if (moba) {
        const uint32_t it = div_by(ok ? v : v_lo, a.by_chunk);
        const int2 item = items_s[it];
        t = item.x * a.chunk + ((ok ? v : v_lo) - it * a.chunk);
        x.mask = item.y;
        ok = ok && t < (uint32_t)len;
      }
      const uint32_t lp = ok ? div_by(t, a.pool.by_page) : 0u;
      x.page = trow[lp];
      x.at = ok ? t - lp * a.pool.by_page.d : ~0u;
      return x;
    };
    // Puts a step's places, from its page entries, where all lanes see them; loads its
    // keys and the scales of the lane's token.  A step behind the last reads the pool's
    // first row over and over: its loads are cheaper than a branch around them, behind
    // which the compiler would wait for every load in flight.
    auto fetch_keys = [&](const Look& x, Keys<NC>& k, Step& s, uint32_t (&voff)[8]) __attribute__((always_inline)) {
      const bool ok = x.at != ~0u && x.page >= 0 && x.page < a.pool.num_pages;
      const uint32_t row = ok ? ((uint32_t)x.page * a.pool.Hkv + kh) * a.pool.P + x.at : 0u;
      off_s[w][lane & 31] = row * pieces;
      s.live = (uint32_t)__ballot(ok);
      s.mask = x.mask;
      s.whole = s.live == ~0u && (!moba || __all(x.mask == heads_mask));
      s.ks = a.pool.ks[row];
      s.vs = a.pool.vs[row];
      wave_lds_sync();
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint8_t* p = a.pool.k + ((uint64_t)off_s[w][16 * t + c16] << 4);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int d = 64 * c + 16 * g;
          k.reg[t][c] = load_once(reinterpret_cast<const u32x4_t*>(p + (d < a.pool.Dp ? d : 0)));
        }
        const u32x4_t o = *reinterpret_cast<const u32x4_t*>(&off_s[w][16 * t + 4 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i) voff[4 * t + i] = o[i];
      }
      wave_lds_sync();
    };
    const int vd = 4 * NC * c16 < a.pool.Dp ? 4 * NC * c16 : 0;
    auto fetch_values = [&](Values<NC>& v, const uint32_t (&voff)[8]) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v.load(j, a.pool.v + ((uint64_t)voff[j] << 4) + vd);
    };
    // Scales of a step, from a lane per token to the scores' layout, and its scores in log2.
    f32x4_t sc[2], vv[2];
    u32x4_t mk[2];
    auto scores = [&](const Keys<NC>& k, const Step& s) __attribute__((always_inline)) {
      if (lane < 32) {
        ks_s[w][lane] = s.ks * a.scale_log2;
        vs_s[w][lane] = s.vs;
        if (moba) mask_s[w][lane] = s.mask;
      }
      wave_lds_sync();
      f32x4_t kk[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        kk[t] = *reinterpret_cast<const f32x4_t*>(&ks_s[w][16 * t + 4 * g]);
        vv[t] = *reinterpret_cast<const f32x4_t*>(&vs_s[w][16 * t + 4 * g]);
        if (moba) mk[t] = *reinterpret_cast<const u32x4_t*>(&mask_s[w][16 * t + 4 * g]);
      }
      wave_lds_sync();
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          u32x4_t lo, hi;
          uint32_t x, y;
          numbers4_16<FMT, DT>(k.reg[t][c][0], x, y); lo[0] = x; lo[1] = y;
          numbers4_16<FMT, DT>(k.reg[t][c][1], x, y); lo[2] = x; lo[3] = y;
          numbers4_16<FMT, DT>(k.reg[t][c][2], x, y); hi[0] = x; hi[1] = y;
          numbers4_16<FMT, DT>(k.reg[t][c][3], x, y); hi[2] = x; hi[3] = y;
          sc[t] = mfma16<DT>(__builtin_bit_cast(u16x8_t, lo), qf[2 * c], sc[t]);
          sc[t] = mfma16<DT>(__builtin_bit_cast(u16x8_t, hi), qf[2 * c + 1], sc[t]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[t][i] *= kk[t][i];
      }
    };
    // The softmax of those scores and their product with the values.
    auto weigh = [&](Values<NC>& v, const Step& s) __attribute__((always_inline)) {
      float p[8], wt[8], top = -INFINITY;
      uint32_t on = 0xff;  // bit j: the lane's head attends its token j
      if (!s.whole) {
        on = ((s.live >> (4 * g)) & 15) | (((s.live >> (16 + 4 * g)) & 15) << 4);
        if (moba) {
          uint32_t takes = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) takes |= ((mk[j >> 2][j & 3] >> my_head) & 1) << j;
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
        for (int t = 0; t < 4 * NC; ++t)
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
      if (!s.whole) {
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
      if (!s.whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool there = (s.live >> (16 * (j >> 2) + 4 * g + (j & 3))) & 1;
#pragma unroll
          for (int d = 0; d < NC; ++d) v.reg[j][d] = there ? v.reg[j][d] : 0;  // never written: may be a NaN's code
        }
      }
#pragma unroll
      for (int d = 0; d < NC; ++d) {
        u32x4_t vt[4];
        v.template operands<FMT>(d, vt);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          acc[4 * d + b] = mfma16<0>(__builtin_bit_cast(u16x8_t, vt[b]), __builtin_bit_cast(u16x8_t, hi), acc[4 * d + b]);
          acc[4 * d + b] = mfma16<0>(__builtin_bit_cast(u16x8_t, vt[b]), __builtin_bit_cast(u16x8_t, lo), acc[4 * d + b]);
        }
      }
    };

    int k = stream;
    if (k < steps) {
      // Loads return in order: the page entries of a step are asked for before the keys
      // and values of the one before it, so that waiting for them waits for nothing else.
      uint32_t voff[8];
      Look now = look(k), next = look(k + streams), after;
      if constexpr (NC <= 2) {
        // two steps in registers: one is on its way while the other is worked on
        Keys<NC> ka, kb;
        Values<NC> va, vb;
        Step sa, sb;
        fetch_keys(now, ka, sa, voff);
        fetch_values(va, voff);
        for (;;) {
          after = look(k + 2 * streams);
          fetch_keys(next, kb, sb, voff);
          fetch_values(vb, voff);
          scores(ka, sa);
          weigh(va, sa);
          k += streams;
          if (k >= steps) break;
          next = look(k + 2 * streams);
          fetch_keys(after, ka, sa, voff);
          fetch_values(va, voff);
          scores(kb, sb);
          weigh(vb, sb);
          k += streams;
          if (k >= steps) break;
        }
      } else {
        // registers for one: its keys make room after the scores, its values after theirs
        Keys<NC> ka;
        Values<NC> va;
        Step sa, sb;
        fetch_keys(now, ka, sa, voff);
        fetch_values(va, voff);
        for (; k < steps; k += streams) {
          scores(ka, sa);
          after = look(k + 2 * streams);
          fetch_keys(next, ka, sb, voff);
          next = after;
          weigh(va, sa);
          fetch_values(va, voff);
          sa = sb;
        }
      }
    }

    // ---- the four waves join; head h of block hb is in waves hb, hb + HB, ...
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) {
      join_m[w][c16] = m;
      join_l[w][c16] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < NC; ++d) {
        const f32x4_t x = {acc[4 * d][i], acc[4 * d + 1][i], acc[4 * d + 2][i], acc[4 * d + 3][i]};
        *reinterpret_cast<f32x4_t*>(&join_o[w][c16][4 * NC * (4 * g + i) + 4 * d]) = x;
      }
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
        const f32x4_t v = *reinterpret_cast<const f32x4_t*>(&join_o[y][h & 15][d]);
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
    left -= n;
    rem += n;
    if (rem == u * (uint32_t)a.scan_mult) { ++si; rem = 0; }
  }
}

// One workgroup per (entry, head) that spans several workgroups of the first launch:
// their partials, weighted by 2^(m_j - m); cols (a power of two) threads of 4 dims each,
// B / cols parts at once, whose sums are added in a fixed order.  An entry without
// tokens gets zeros and -inf.
template <int DT, int B>
__global__ __launch_bounds__(B) void join_kernel(AttnArgs a, int wgs, int cols, int per_entry) {
  __shared__ float weight[kMaxWgs];
  __shared__ float red[2][B / 64];
  __shared__ __attribute__((aligned(16))) f32x4_t sums[B / 64][64];
  const int hpe = 16 * a.HB, e = blockIdx.x / per_entry, h = blockIdx.x % per_entry;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int r = e / a.per_row, kh = (e % a.per_row) / a.NHB, blk = e % a.NHB;
  if (h >= a.G - blk * hpe) return;
  const int D = a.pool.D;
  const int si = e / a.scan_mult;
  const uint32_t T = a.start[a.scan_n], s0 = a.start[si], u = (a.start[si + 1] - s0) / a.scan_mult;
  const int64_t row = (int64_t)r * a.Hq + kh * a.G + blk * hpe + h;
  if (u == 0) {
    for (int d = tid; d < D; d += B) a.out[row * D + d] = 0;
    if (tid == 0) a.lse[row] = -INFINITY;
    return;
  }
  const uint32_t W = min((uint32_t)wgs, T), from = s0 + (e % a.scan_mult) * u;
  const Deal deal(T, W);
  const uint32_t w0 = deal.owner(from), w1 = deal.owner(from + u - 1), parts = w1 - w0 + 1;
  if (parts == 1) return;  // written by that workgroup
  // workgroup x's partial of this entry: its first segment's, if its run begins within
  // the entry (all but w0's do), else its last one's
  const int64_t slot0 = ((int64_t)2 * w0 + (deal.first(w0) < from ? 1 : 0)) * hpe + h;
  auto slot = [&](uint32_t j) { return j == 0 ? slot0 : (int64_t)2 * (w0 + j) * hpe + h; };
  float top = -INFINITY;
  for (uint32_t j = tid; j < parts; j += B) top = fmaxf(top, a.part_ml[2 * slot(j)]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if (lane == 0) red[0][w] = top;
  __syncthreads();
  for (int x = 0; x < B / 64; ++x) top = fmaxf(top, red[0][x]);
  float z = 0.0f;
  for (uint32_t j = tid; j < parts; j += B) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * slot(j));
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
  const int c = tid & (cols - 1), d = 4 * c, groups = B / cols;
  const int at = d < D ? d : 0;  // columns behind D repeat the first
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (uint32_t j = tid / cols; j < parts; j += groups) {
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.part_o + slot(j) * D + at);
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
  const float f = z == 0.0f ? 0.0f : 1.0f / z;
  *reinterpret_cast<uint2*>(a.out + row * D + d) =
      make_uint2(pack2<DT>(o[0] * f, o[1] * f), pack2<DT>(o[2] * f, o[3] * f));
  if (d == 0) a.lse[row] = z == 0.0f ? -INFINITY : (top + __log2f(z)) * kLn2;
}

// Shape of a call: blocks of heads, entries, workgroups, and what its workspace holds.
struct Shape {
  int G, HB, NHB, max_items, wgs;
  int64_t entries, items_at, tokens_at, start_at, part_o_at, part_ml_at, bytes;
};
Shape shape_of(int Nq, int Hq, int Hkv, int D, int slots, int chunk, int max_length) {
  Shape s;
  s.G = Hq / Hkv;
  s.HB = s.G > 16 ? 2 : 1;
  s.NHB = (s.G + 16 * s.HB - 1) / (16 * s.HB);
  s.entries = (int64_t)Nq * Hkv * s.NHB;
  s.max_items = std::min(s.G, 16 * s.HB) * slots;
  // as many workgroups as the card holds at once, but no more than there can be units
  const int per_cu = D > 64 ? 2 : 3;
  const int64_t longest = slots > 0 ? std::min<int64_t>((int64_t)s.max_items * chunk, max_length) : max_length;
  const int64_t units = s.entries * ((longest + kUnit - 1) / kUnit);
  s.wgs = (int)std::min<int64_t>(256 * per_cu, (units + 7) / 8 * 8);
  if (s.wgs < 8) s.wgs = 8;
  auto take = [&](int64_t n) { const int64_t at = s.bytes; s.bytes += (n + 255) / 256 * 256; return at; };
  s.bytes = 0;
  s.items_at = take(slots > 0 ? s.entries * s.max_items * 8 : 0);
  s.tokens_at = take(slots > 0 ? s.entries * 4 : 0);
  s.start_at = take((std::max<int64_t>(slots > 0 ? s.entries : Nq, 1) + 1) * 4);
  const int64_t rows = 2ll * s.wgs * 16 * s.HB;
  s.part_o_at = take(rows * D * 4);
  s.part_ml_at = take(rows * 8);
  return s;
}

template <int DT, int FMT> void launch_attend(const AttnArgs& a, int wgs, hipStream_t st) {
  const dim3 grid(wgs), block(256);
  if (a.pool.Dp <= 64) hipLaunchKernelGGL((attend_kernel<DT, FMT, 1>), grid, block, 0, st, a);
  else if (a.pool.Dp <= 128) hipLaunchKernelGGL((attend_kernel<DT, FMT, 2>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((attend_kernel<DT, FMT, 4>), grid, block, 0, st, a);
}

// Few joins have many parts each: wide workgroups then.
template <int DT> void launch_join(const AttnArgs& a, unsigned joins, int wgs, int cols, int per_entry, hipStream_t st) {
  if (joins <= 256) hipLaunchKernelGGL((join_kernel<DT, 1024>), dim3(joins), dim3(1024), 0, st, a, wgs, cols, per_entry);
  else hipLaunchKernelGGL((join_kernel<DT, 256>), dim3(joins), dim3(256), 0, st, a, wgs, cols, per_entry);
}

}  // namespace

extern "C" int64_t moba_hip_quantized_attention_work(int Nq, int Hq, int Hkv, int D, int slots, int chunk,
                                                     int max_length) {
  if (Nq < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || D < 8 || D > 256 || slots < 0 || slots > kMaxSlots ||
      (slots > 0 && chunk < 1) || max_length < 1)
    return -1;
  return shape_of(Nq, Hq, Hkv, D, slots, chunk, max_length).bytes;
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
  if (!(scale >= 0x1p-126f && scale < 1e30f)) { moba_set_error("quantized_attention: scale must be in [2^-126, 1e30]"); return MOBA_ERR_ARG; }
  if (max_length < 1) { moba_set_error("quantized_attention: max_length must be positive"); return MOBA_ERR_ARG; }
  if ((selected != nullptr) != (slots > 0) || slots > kMaxSlots || (selected != nullptr && chunk < 1)) { moba_set_error("quantized_attention: selected chunks need 1 to 16 slots and a chunk size"); return MOBA_ERR_ARG; }
  if ((((uintptr_t)q | (uintptr_t)out | (uintptr_t)work) & 15) || work == nullptr) { moba_set_error("quantized_attention: q, out and work must be 16-byte aligned"); return MOBA_ERR_ARG; }
  max_length = (int)std::min<int64_t>(max_length, (int64_t)table_width * page_size);
  chunk = std::min(chunk, max_length);  // a longer one ends where the row does
  const Shape s = shape_of(Nq, Hq, Hkv, D, slots, chunk, max_length);
  // units, tokens and workgroups of the second launch are counted in 31 bits
  if (max_length > 0x7fffff00 || s.entries * ((max_length + kUnit - 1ll) / kUnit) >= 1ll << 31 ||
      s.entries * 16 * s.HB >= 1ll << 31) {
    moba_set_error("quantized_attention: more than 2^31 tokens of a row, units of 128 tokens or heads");
    return MOBA_ERR_ARG;
  }
  char* p = (char*)work;
  a.q = (const uint16_t*)q;
  a.Hq = Hq; a.G = s.G; a.HB = s.HB; a.NHB = s.NHB; a.per_row = Hkv * s.NHB;
  a.q_seq = q_seq; a.lengths = lengths; a.length_add = length_add; a.max_length = max_length;
  a.selected = selected; a.slots = slots; a.chunk = chunk; a.max_items = s.max_items;
  a.by_chunk = fast_div(std::max(1, chunk)); a.by_d4 = fast_div(D / 4);
  a.items = (int2*)(p + s.items_at); a.tokens = (int*)(p + s.tokens_at);
  a.scan_n = selected != nullptr ? (int)s.entries : Nq;
  a.scan_mult = selected != nullptr ? 1 : a.per_row;
  a.start = (uint32_t*)(p + s.start_at);
  a.scale_log2 = scale * kLog2e;
  a.part_o = (float*)(p + s.part_o_at); a.part_ml = (float*)(p + s.part_ml_at);
  a.out = (uint16_t*)out; a.lse = lse;
  hipStream_t st = (hipStream_t)stream;
  if (selected != nullptr) hipLaunchKernelGGL(union_kernel, dim3((unsigned)s.entries), dim3(64), 0, st, a);
  if (dtype == 0) { if (format == 0) launch_attend<0, 0>(a, s.wgs, st); else launch_attend<0, 1>(a, s.wgs, st); }
  else { if (format == 0) launch_attend<1, 0>(a, s.wgs, st); else launch_attend<1, 1>(a, s.wgs, st); }
  int cols = 16;
  while (cols * 4 < D) cols *= 2;
  const int per_entry = std::min(s.G, 16 * s.HB);
  const unsigned joins = (unsigned)(s.entries * per_entry);
  if (dtype == 0) launch_join<0>(a, joins, s.wgs, cols, per_entry, st);
  else launch_join<1>(a, joins, s.wgs, cols, per_entry, st);
  return moba_launch_status("quantized_attention");
}
