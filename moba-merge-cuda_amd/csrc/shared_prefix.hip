// Attention of a batch whose sequences share long prefixes, on a paged cache.
//
// Query row r attends the tokens [0, P) of the prefix slot it shares and then
// the tokens [0, L_r) of its own slot:
//   s_j = scale q.k_j,  out = sum_j e^{s_j - m} v_j / z,  z = sum_j e^{s_j - m},
//   lse = m + ln z,     m = max_j s_j over both.
// The keys are cut into ranges, and every range is one work item of all the
// rows that attend it (prefix: all rows of the batch that share it; own tokens:
// the rows of one slot), times the q heads of a kv head: a block of up to 128
// (row, head) pairs against the range's K/V, read once for the block.  An item
// leaves (O, m, z) of its range in fp32; merge_kernel joins a row's ranges in
// their order.  Results do not depend on timing.
//
// Scores, softmax and sums are fp32.  Two roundings to 16 bits are the matrix
// units' price: the weights e^{s - m} before their product with V, and the result.
// A weight is off by at most half a step of its own, 2^-8 (bf16) or 2^-11 (fp16),
// its sum z takes it unrounded.  fp16 weights reach from 2^7 or more for the
// largest of a wave's keys to 2^15 (m lies below the maximum by that), so that
// only what is 2^21 below the largest is subnormal, off by 2^-32 of the largest:
// a flat tail of 2^17 keys behind one strong key is right to 2^-15.
//
// What bounds it: with many pairs to a block the products and the exponentials,
// which share a SIMD's issue slots (D 128, 1024 rows behind 16K tokens: matrix
// units busy 57% of the cycles, vector instructions 57%, together 89%, at 1.65
// GHz, to which the chip's power limit takes the clock); with few the reads of
// K and V; with few tokens the chain launch, page entries, keys, values, partials
// and the second launch.
#include <type_traits>

#include "common.h"
#include "../../include/moba_hip.h"

using namespace moba;

namespace {

// One work item (the plan's int32 record).
struct Item {
  int row_at;   // its segment's first entry of `rows`
  int m0;       // first (row, q head of the kv head) pair of the block: row m / G
  int n_m;      // pairs of the block; 0: none; -1: each wave has the item of its
                // own at row_at + wave
  int slot;     // page-table row of the keys
  int kh;
  int split;    // split | splits << 16
  int length;   // tokens of the segment; -1: each row's own length
  int row;      // the row of the block's pairs; -1: several
};

struct SharedArgs {
  const uint16_t *q, *kc, *vc;
  int Hq, Hkv, D, G;
  float scale_log2;
  int num_pages, P, W;
  uint32_t pool_bytes;      // of k_cache; 0: 4 GiB or more
  const int* table;
  const int* lengths;       // own tokens of each row
  int length_add, max_length;  // own length of a row: lengths[row] + length_add, cut
  const Item* items;
  const int* rows;
  const int *prefix_at, *own_at, *n_part;  // per row: first partials, ranges in all
  float* part_o;
  float2* part_ml;
};

// 16 bytes per lane straight into LDS (lane l's at LDS address lds + 16 l), from
// a buffer or from any address; ordered by the caller as dma_lds16.
MOBA_DEV void dma_buffer16(__amdgpu_buffer_rsrc_t r, uint32_t lds, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds), "v"(voff), "s"(r) : "memory", "m0");
}
MOBA_DEV void dma_global16(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds), "v"(p) : "memory", "m0");
}
// s_waitcnt vmcnt(N) for any N, and nothing moves across it.
template <int N> MOBA_DEV void landed() {
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14);
  asm volatile("" ::: "memory");
}
// This wave's LDS reads are complete.
MOBA_DEV void lds_read_done() {
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("" ::: "memory");
}

// Sizes of a head dim's kernel.
template <int ND> struct Dims {
  static constexpr int DP = ND <= 64 ? 64 : ND <= 128 ? 128 : 256;  // row of the LDS layouts
  static constexpr int NKS = ND / 16, NDB = ND / 32, NB = DP / 8;
  static constexpr int KEYS = DP <= 64 ? 64 : 32;   // keys of a tile that four waves share
  static constexpr int TILE = KEYS * DP;
  static constexpr int OWN = DP <= 64 ? 32 : 16;    // keys of a tile that a wave has alone
  // LDS: stages of shared K and V tiles, or a K and a V tile per wave; the
  // pool's token of up to CAP keys; flags.  Three workgroups share a CU up to 128
  // dims, two above.
  static constexpr int STAGES = DP <= 128 ? 3 : 2, CAP = 1024;
  static constexpr int TILES = STAGES * TILE * 2 * 2;
  static_assert(4 * 2 * OWN * DP * 2 <= TILES && 4 * 3 * 4 * 64 * 16 <= TILES && CAP * 4 >= 4 * 64 * 8, "LDS");
  static constexpr int TOK = TILES, FLAGS = TOK + CAP * 4, LDS = FLAGS + 16;
  static constexpr int WAVES = ND <= 128 ? 3 : 2;   // per SIMD
};

// Where a key's row of the pool is: its byte offset below 4 GiB (NEAR), else
// its token.  A key of no token, or of an unmapped page, loads zeros, so that a
// weight of 0 meets no NaN: its offset lies outside the buffer resource.
constexpr uint32_t kNowhere = 0xffff0000u;
__device__ __attribute__((aligned(16))) const uint16_t g_zero[8] = {0};

// The K and V rows of a kv head in the pool.
template <bool NEAR> struct Rows {
  __amdgpu_buffer_rsrc_t k, v;
  const char *kp, *vp;
  uint32_t row_bytes;
  MOBA_DEV Rows(const SharedArgs& a, int kh) {
    const uint32_t head = (uint32_t)(kh * a.D * 2);
    kp = (const char*)a.kc + head;
    vp = (const char*)a.vc + head;
    row_bytes = (uint32_t)(a.Hkv * a.D * 2);
    if constexpr (NEAR) {
      k = make_rsrc(kp, a.pool_bytes - head);
      v = make_rsrc(vp, a.pool_bytes - head);
    }
  }
  MOBA_DEV uint32_t place(uint32_t token) const { return NEAR ? token * row_bytes : token; }
  // 64 lanes' 16-byte blocks, `byte` into the row at `at`, to LDS address lds
  template <bool V> MOBA_DEV void bring(uint32_t at, uint32_t byte, uint32_t lds) const {
    if constexpr (NEAR) {
      dma_buffer16(V ? v : k, lds, at + byte);
    } else {
      const char* p = (V ? vp : kp) + (uint64_t)at * row_bytes + byte;
      dma_global16(at != kNowhere ? p : (const char*)g_zero, lds);
    }
  }
};

// A row's own length.
MOBA_DEV int own_length(const SharedArgs& a, int row) {
  return (int)max(0ll, min((long long)a.lengths[row] + a.length_add, (long long)a.max_length));
}
// What a lane knows of its (row, q head) pair.
struct Pair {
  int row, h, limit;   // limit: tokens of the segment that the row attends
  int64_t part;        // its partial
  bool valid;
};
// alike: the tokens that all the rows attend, -1 if they differ.
MOBA_DEV Pair pair_of(const SharedArgs& a, const Item& x, int m, int alike) {
  Pair p;
  p.valid = m < x.n_m;
  const int i = x.m0 + min(m, x.n_m - 1), r = i / a.G;
  p.h = x.kh * a.G + i - r * a.G;
  p.row = x.row >= 0 ? x.row : a.rows[x.row_at + r];
  p.limit = alike >= 0 ? alike : own_length(a, p.row);
  p.part = ((int64_t)(x.length < 0 ? a.own_at : a.prefix_at)[p.row] + (x.split & 0xffff)) * a.Hq + p.h;
  return p;
}
// Of a segment or of one row: a scalar load at most.
MOBA_DEV int alike_of(const SharedArgs& a, const Item& x) {
  return x.length >= 0 ? x.length : x.row >= 0 ? own_length(a, x.row) : -1;
}
// Longest and shortest row of the lanes' 32 pairs, the same in every lane.
MOBA_DEV int longest(int limit) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) limit = max(limit, __shfl_xor(limit, o, 64));
  return __builtin_amdgcn_readfirstlane(limit);
}
MOBA_DEV int shortest(const Pair& p, int alike) {
  if (alike >= 0) return alike;
  int limit = p.valid ? p.limit : 0x7fffffff;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) limit = min(limit, __shfl_xor(limit, o, 64));
  return __builtin_amdgcn_readfirstlane(limit);
}
// The keys [lo, hi) of an item's range: whole groups of 64 but for the last.
MOBA_DEV void range_of(const Item& x, int length, int& lo, int& hi) {
  length = max(length, 0);
  const int split = x.split & 0xffff, splits = (uint32_t)x.split >> 16;
  const int per = (int)((length + 64ll * splits - 1) / (64 * splits)) * 64;
  lo = (int)min((int64_t)length, (int64_t)split * per);
  hi = (int)min((int64_t)length, (int64_t)lo + per);
}
// The page-table entry of a key (of the last key behind hi).
MOBA_DEV int entry_of(const SharedArgs& a, int slot, int key, int hi) {
  return a.table[(int64_t)slot * a.W + min(key, hi - 1) / a.P];
}
// Looks up the keys [k0, min(k0 + CAP, hi)) with WIDTH threads (and fills to a
// multiple of WIDTH with kNowhere), the first WIDTH from the entries `first`.
// Returns whether a page of the wave's keys is unmapped.
template <bool NEAR, int CAP, int WIDTH>
MOBA_DEV bool look_up(const SharedArgs& a, const Rows<NEAR>& rows, int slot, int k0, int hi,
                      int first, int thread, uint32_t* tok) {
  const int n = min(CAP, hi - k0);
  bool holes = false;
  for (int i0 = 0; i0 < n; i0 += WIDTH) {
    const int at = k0 + i0 + thread, page = i0 ? entry_of(a, slot, at, hi) : first;
    const int key = min(at, hi - 1), in_page = key - key / a.P * a.P;
    const bool mapped = page >= 0 && page < a.num_pages;
    tok[i0 + thread] = (at < hi) & mapped ? rows.place((uint32_t)page * a.P + in_page) : kNowhere;
    holes |= !mapped;
  }
  return __any(holes);
}
// After a barrier: whether any wave saw one.
MOBA_DEV bool any_hole(const int* flags) {
  const int4 f = *reinterpret_cast<const int4*>(flags);
  return __builtin_amdgcn_readfirstlane(f.x | f.y | f.z | f.w) != 0;
}

template <int NDB>
MOBA_DEV void store_partial(const SharedArgs& a, int64_t part, const f32x16_t (&o)[NDB], float m,
                            float l, int hh) {
  float* po = a.part_o + part * a.D;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = db * 32 + 8 * j + 4 * hh;
      if (d < a.D)
        *reinterpret_cast<f32x4_t*>(po + d) =
            (f32x4_t){o[db][4 * j], o[db][4 * j + 1], o[db][4 * j + 2], o[db][4 * j + 3]};
    }
  if (hh == 0) a.part_ml[part] = make_float2(m, l);
}

// A lane's pair's running softmax: reference (log2 domain), sum of this lane's
// keys, and what the next tile needs of the reference.  The reference is set
// kBelow below the largest score and stays while the scores are at most kSlack
// above that one: weights, which are relative to it, reach 2^8 in bf16 and 2^15
// in fp16 (whose largest value is 65504), where small weights need the room.
struct Running {
  float m = -INFINITY, l = 0.0f;
  float nm = 0.0f;            // -m; 0 while nothing was attended: weights of
                              // 0, not of exp2(-inf + inf)
  float limit = -INFINITY;    // scores above move the reference
};
constexpr float kSlack = 8.0f;
template <int DT> constexpr float kBelow = DT == 0 ? 0.0f : 7.0f;

// Maximum over the lanes l and l + 32.
MOBA_DEV float max_halves(float x) {
  uint32_t a = __float_as_uint(x), b = a;
  swap_halves(a, b);
  return fmaxf(__uint_as_float(a), __uint_as_float(b));
}

// One tile's scores (the first NR registers of each block) into the running
// softmax; returns the 16-bit weights as operands of the product with V.
template <int DT, int NKB, int NR, int NDB>
MOBA_DEV void softmax_step(const f32x16_t (&s)[NKB], float c2, Running& run, f32x16_t (&o)[NDB],
                           u16x8_t (&pv)[NKB][NR / 8]) {
  float mx = -INFINITY;
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
    for (int r = 0; r < NR; ++r) mx = fmaxf(mx, s[kb][r]);
  mx = max_halves(mx) * c2;
  const bool up = mx > run.limit;
  if (__any(up)) [[unlikely]] {
    const float mn = up ? mx - kBelow<DT> : run.m;
    const float alpha = up ? fast_exp2(run.m - mn) : 1.0f;
    run.l *= alpha;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
    run.m = mn;
    run.nm = mn == -INFINITY ? 0.0f : -mn;
    run.limit = mn + (kBelow<DT> + kSlack);
    __builtin_amdgcn_sched_barrier(0);
  }
  float ps = 0.0f;
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb) {
    float p[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      p[r] = fast_exp2(fmaf(s[kb][r], c2, run.nm));
      ps += p[r];
    }
#pragma unroll
    for (int t = 0; t < NR / 8; ++t) pv[kb][t] = pack8<DT>(p + 8 * t);
  }
  run.l += ps;
}

// Scores of keys behind `left` (counted from the tile's first) or, with holes,
// of unmapped pages: -inf.  tok: the tile's keys.
template <int NKB, int NR>
MOBA_DEV void mask_scores(f32x16_t (&s)[NKB], int left, const uint32_t* tok, int hh) {
  left = (int)opaque(left - 4 * hh);  // a lane's keys are 4 hh + constants: none to keep in registers
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
    for (int j = 0; j < NR / 4; ++j) {
      const int k = kb * 32 + 8 * j + 4 * hh;
      const u32x4_t t = *reinterpret_cast<const u32x4_t*>(tok + k);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[kb][4 * j + i] = (kb * 32 + 8 * j + i < left) & (t[i] != kNowhere) ? s[kb][4 * j + i] : -INFINITY;
    }
}

// N products in order, what each reads from LDS (in READS instructions) sent out
// before the one two or three before it.  FIXED: exactly so; the compiler, left to
// it, sends a read out right before its product where registers are short (1024
// rows of 256 dims behind 8K tokens: 176 us, 162 so; two before 163, four 172), and
// at 128 dims does 1% better from the wish alone (1024 rows behind 16K: 299 us as it
// orders them, 296 so).
template <int N, int READS, bool FIXED, class Load, class Use> MOBA_DEV void in_order(Load load, Use use) {
  constexpr int AHEAD = N < 3 ? N : FIXED ? 3 : 2;
  u16x8_t f[N];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) f[i] = load(i);
  if constexpr (FIXED) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    use(i, f[i]);
    if (i + AHEAD < N) f[i + AHEAD] = load(i + AHEAD);
    if constexpr (FIXED) __builtin_amdgcn_sched_barrier(0);
  }
  if constexpr (!FIXED) {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * READS, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      if (i + AHEAD < N) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
  }
}
// The i-th of N fragments in an order where those a constant apart (PER of
// them) follow each other: one address in a register serves them.
template <int N, int PER> constexpr int by_address(int i) {
  constexpr int G = (N + PER - 1) / PER, LONG = N - PER * (G - 1);  // LONG runs of G, then of G - 1
  if (G == 1) return i;
  const int j = i - G * LONG;
  return j < 0 ? i / G + i % G * PER : LONG + j / (G - 1) + j % (G - 1) * PER;
}
// First byte of the 16-byte block that lane `lane` brings in a load of 64
// blocks of the swizzled layout whose first row is row0: physical block lane %
// NB of row row0 + lane / NB.  The swizzle's bit reversal takes row0 and lane /
// NB apart, which share no bits.
template <int DP> MOBA_DEV uint32_t block_byte(uint32_t lane, uint32_t row0) {
  constexpr uint32_t NB = DP / 8, NBM = (uint32_t)swz_nbm<DP>();
  const uint32_t f = (__builtin_bitreverse32(lane / NB) ^ __builtin_bitreverse32(row0)) >> 28;
  return ((lane % NB) ^ (f & NBM)) * 16;
}

// A weight of 0 times an infinite or NaN value is NaN, which a row must not get
// from a key behind its own length that another row of the block attends.  In
// tiles with such keys, values that are not finite are replaced by zeros; where
// that happened, the tiles are read again after the others, and every row gets
// what it attends of them: +inf or -inf if there is only the one, else NaN.
// Only kernels of plans where several rows have one own slot (UNEVEN) do this: it
// takes registers and branches from all their items (64 rows behind 32K tokens:
// 114 us without, 123 with).
//
// 0xffff for each of a word's two values that is not finite; for each that has
// no mantissa bits (no carries: a half's bits plus 0x7fff stay below 2^16).
MOBA_DEV uint32_t zero_halves(uint32_t w) {
  const uint32_t z = ~(w + 0x7fff7fffu) & 0x80008000u;
  return z | (z - (z >> 15));
}
template <int DT> MOBA_DEV uint32_t not_finite(uint32_t w) {
  return zero_halves(~w & (DT == 0 ? 0x7f807f80u : 0x7c007c00u));
}
template <int DT> MOBA_DEV uint32_t no_mantissa(uint32_t w) {
  return zero_halves(w & (DT == 0 ? 0x007f007fu : 0x03ff03ffu));
}
// Zeros in the place of what is not finite in the wave's share (from thread
// `thread` of WIDTH) of a tile of N values; whether there was any.
template <int DT, int N, int WIDTH> MOBA_DEV bool odd_in(uint16_t* V, int thread) {
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < N / (8 * WIDTH); ++i) {
    u32x4_t* at = reinterpret_cast<u32x4_t*>(V) + i * WIDTH + thread;
    u32x4_t v = *at;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t b = not_finite<DT>(v[k]);
      bad |= b;
      v[k] &= ~b;
    }
    *at = v;
  }
  return __any(bad != 0);
}
// o += what is not finite among the values of a tile of NG groups of 16 keys,
// for the lane's row, which attends the keys before `left`.
template <int DT, int DP, int NDB, int NG>
MOBA_DEV void add_odd(const uint16_t* V, int lane, int left, const uint32_t* tok, f32x16_t (&o)[NDB]) {
  constexpr uint32_t one = DT == 0 ? 0x3f803f80u : 0x3c003c00u;
  const int hh = lane >> 5;
  u32x4_t on[NG];  // 1 for the keys that the row attends, laid out as weights
#pragma unroll
  for (int g = 0; g < NG; ++g)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int k = g * 16 + 8 * j + 4 * hh;
      const u32x4_t t = *reinterpret_cast<const u32x4_t*>(tok + k);
      uint32_t m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = (k + i < left) & (t[i] != kNowhere) ? one : 0;
      on[g][2 * j] = (m[0] & 0xffffu) | (m[1] << 16);
      on[g][2 * j + 1] = (m[2] & 0xffffu) | (m[3] << 16);
    }
  const uint32_t t0 = swz_tr_base<DP>(lane, 0), t1 = swz_tr_base<DP>(lane, 1);
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    f32x16_t odd = zero16(), sign = zero16();
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const uint32_t ro = g * 16 * DP * 2;
      const u32x4_t v = __builtin_bit_cast(
          u32x4_t, lds_tr8(V, ro + swz_tr<DP>(opaque(t0), db), ro + swz_tr<DP>(opaque(t1), db)));
      u32x4_t c, s;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t bad = not_finite<DT>(v[k]);
        c[k] = bad & one;
        s[k] = bad & no_mantissa<DT>(v[k]) & ((v[k] & 0x80008000u) | one);
      }
      odd = mfma32<DT>(__builtin_bit_cast(u16x8_t, c), __builtin_bit_cast(u16x8_t, on[g]), odd);
      sign = mfma32<DT>(__builtin_bit_cast(u16x8_t, s), __builtin_bit_cast(u16x8_t, on[g]), sign);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float bad = fabsf(sign[r]) == odd[r] ? copysignf(INFINITY, sign[r]) : NAN;
      o[db][r] += odd[r] != 0.0f ? bad : 0.0f;
    }
    __builtin_amdgcn_sched_barrier(0);  // a block at a time
  }
}

template <int NKS> MOBA_DEV void load_query(const SharedArgs& a, const Pair& p, int hh, u16x8_t (&qf)[NKS]) {
  const uint16_t* q = a.q + ((int64_t)p.row * a.Hq + p.h) * a.D;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const int d = ks * 16 + hh * 8;
    const u16x8_t v = ld8(q + (d < a.D ? d : 0));
    qf[ks] = d < a.D ? v : zero8();
  }
}

// More than 32 pairs: every wave has 32 of them, and the four share tiles of
// KEYS keys in STAGES LDS stages: while one is in use, the loads of the others are
// in flight.  S^T = K Q^T and O^T += V^T P^T: a lane holds one pair's column of
// both, so that its maximum and sum take one exchange with lane + 32 and the
// weights are the second product's operand where they are.  128 pairs: K and V
// are read from L2 once for 128 x 4 D operations a key; 64 rows to a wave spilled
// at 64 dims and gave 2% at 128.  Bound by products and exponentials: 1024 rows
// of 4 heads a kv head behind 16K tokens, D 128, 296 us, 0.93 PFLOP/s.
template <int DT, int ND, bool NEAR, bool UNEVEN>
MOBA_DEV void wide_item(const SharedArgs& a, const Item& x, char* smem) {
  typedef Dims<ND> C;
  constexpr int DP = C::DP, NKS = C::NKS, NDB = C::NDB, KEYS = C::KEYS, NKB = KEYS / 32;
  constexpr int TILE = C::TILE, NB = C::NB, NDMA = KEYS * NB / 256;
  constexpr int STAGES = C::STAGES;
  uint16_t* Ks = (uint16_t*)smem;   // [STAGES][TILE], then V
  uint32_t* tok = (uint32_t*)(smem + C::TOK);
  int* flags = (int*)(smem + C::FLAGS);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 31, hh = lane >> 5, D = a.D;

  const int alike = alike_of(a, x);
  const Pair p = pair_of(a, x, wave * 32 + qi, alike);
  int length = alike, block_least = 0x7fffffff;
  if (length < 0) {  // the block's longest and shortest row
    const int mine = longest(p.limit);
    if (lane == 0) flags[wave] = mine;
    lds_barrier();
    length = max(max(flags[0], flags[1]), max(flags[2], flags[3]));
    lds_barrier();
    if constexpr (UNEVEN) {
      const int least = shortest(p, alike);
      if (lane == 0) flags[wave] = least;
      lds_barrier();
      block_least = min(min(flags[0], flags[1]), min(flags[2], flags[3]));
      lds_barrier();
    }
  }
  int lo, hi;
  range_of(x, length, lo, hi);
  if (lo >= hi) {
    if (p.valid && hh == 0) a.part_ml[p.part] = make_float2(-INFINITY, 0.0f);
    return;
  }
  const Rows<NEAR> rows(a, x.kh);
  int first = entry_of(a, x.slot, lo + tid, hi);
  u16x8_t qf[NKS];
  load_query<NKS>(a, p, hh, qf);

  f32x16_t oacc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) oacc[db] = zero16();
  Running run;
  const bool idle = wave * 32 >= x.n_m;
  const int wlim = min(shortest(p, alike), hi);
  const uint32_t kbase0 = swz_b128_base<DP>(lane);
  const uint32_t trb0 = swz_tr_base<DP>(lane, 0), trb1 = swz_tr_base<DP>(lane, 1);

  // wave w brings the 64-block loads n * 4 + w of a tile; where a tile's rows
  // are is read one tile before
  const uint32_t lds0 = lds_addr(smem) + wave * 1024;
  const uint32_t byte0 = block_byte<DP>(lane, wave * (64 / NB));
  // (above 128 dims recomputed at each load: registers are short there)
  auto byte = [&](int n) { return (DP > 128 ? opaque(byte0) : byte0) ^ block_byte<DP>(0, n * 4 * (64 / NB)); };
  uint32_t at[NDMA];
  bool mine[NDMA];
#pragma unroll
  for (int n = 0; n < NDMA; ++n) mine[n] = byte(n) < (uint32_t)D * 2;
  auto places = [&](int it) {
#pragma unroll
    for (int n = 0; n < NDMA; ++n) at[n] = tok[it * KEYS + (n * 4 + wave) * (64 / NB) + lane / NB];
  };
  auto dma = [&](auto stage) {
    const uint32_t lds = lds0 + decltype(stage)::value * (TILE * 2);
#pragma unroll
    for (int n = 0; n < NDMA; ++n)
      if (mine[n]) {
        rows.template bring<false>(at[n], byte(n), lds + n * 4096);
        rows.template bring<true>(at[n], byte(n), lds + STAGES * TILE * 2 + n * 4096);
      }
  };
  auto tile = [&](auto stage, int it, int kt0, bool holes) {
    const uint16_t *Kb = Ks + decltype(stage)::value * TILE, *Vb = Kb + STAGES * TILE;
    const uint32_t kq = opaque(kbase0), t0 = opaque(trb0), t1 = opaque(trb1);
    f32x16_t sacc[NKB];
    wave_prio<1>();
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) sacc[kb] = zero16();
    in_order<NKB * NKS, 1, (DP > 128)>(
        [&](int i) {
          return lds8(Kb, i / NKS * 32 * DP * 2 + swz_b128<DP>(kq, by_address<NKS, 8>(i % NKS)));
        },
        [&](int i, u16x8_t k) {
          sacc[i / NKS] = mfma32<DT>(k, qf[by_address<NKS, 8>(i % NKS)], sacc[i / NKS]);
        });
    wave_prio<0>();
    if (kt0 + KEYS > wlim || holes)
      mask_scores<NKB, 16>(sacc, min(p.limit, hi) - kt0, tok + it * KEYS, hh);
    u16x8_t pv[NKB][2];
    softmax_step<DT, NKB, 16, NDB>(sacc, a.scale_log2, run, oacc, pv);
    wave_prio<1>();
    in_order<NDB * NKB * 2, 2, (DP > 128)>(
        [&](int i) {
          const uint32_t ro = i % (2 * NKB) * 16 * DP * 2;
          const int db = by_address<NDB, 4>(i / (2 * NKB));
          return lds_tr8(Vb, ro + swz_tr<DP>(t0, db), ro + swz_tr<DP>(t1, db));
        },
        [&](int i, u16x8_t v) {
          const int db = by_address<NDB, 4>(i / (2 * NKB));
          oacc[db] = mfma32<DT>(v, pv[i % (2 * NKB) / 2][i % 2], oacc[db]);
        });
    wave_prio<0>();
  };

  // Looks up the keys from k0 on; returns whether a page of theirs is unmapped.
  auto chunk = [&](int k0) {
    const bool mine = look_up<NEAR, C::CAP, 256>(a, rows, x.slot, k0, hi, first, tid, tok);
    if (lane == 0) flags[wave] = mine;
    lds_barrier();
    landed<0>();  // what the compiler has in flight: it must not wait for it below
    return any_hole(flags);
  };
  bool odd = false;
  for (int k0 = lo; k0 < hi; k0 += C::CAP) {
    if (k0 > lo) {
      lds_barrier();  // the tokens and tiles before are read
      first = entry_of(a, x.slot, k0 + tid, hi);
    }
    const bool holes = chunk(k0);
    const int ntiles = (min(hi - k0, C::CAP) + KEYS - 1) / KEYS;
    // the loads of a tile: 2 NDMA, issued STAGES - 1 tiles ahead
    auto step = [&](auto stage, int it) {
      constexpr int S = decltype(stage)::value;
      if (it + 1 < ntiles) landed<(STAGES - 2) * 2 * NDMA>();  // this wave's part of tile `it`
      else landed<0>();
      lds_barrier();  // everyone's, and tile it - 1 is read
      if (it + STAGES - 1 < ntiles) {
        dma(std::integral_constant<int, (S + STAGES - 1) % STAGES>{});
        places(min(it + STAGES, ntiles - 1));
      }
      const int kt0 = k0 + it * KEYS;
      if constexpr (UNEVEN)
        if (kt0 + KEYS > block_least) {  // rows of unlike lengths end in this tile
          odd |= odd_in<DT, TILE, 256>(Ks + (STAGES + S) * TILE, tid);
          lds_barrier();
        }
      if (!idle) tile(stage, it, kt0, holes);
    };
    places(0);
    dma(std::integral_constant<int, 0>{});
    if constexpr (STAGES > 2) {
      places(min(1, ntiles - 1));
      if (ntiles > 1) dma(std::integral_constant<int, 1>{});
    }
    places(min(STAGES - 1, ntiles - 1));
    for (int it = 0; it < ntiles; it += STAGES) {
      step(std::integral_constant<int, 0>{}, it);
      if (it + 1 < ntiles) step(std::integral_constant<int, 1>{}, it + 1);
      if constexpr (STAGES > 2)
        if (it + 2 < ntiles) step(std::integral_constant<int, 2>{}, it + 2);
    }
  }
  if (UNEVEN && alike < 0) {
    lds_barrier();
    if (lane == 0) flags[wave] = odd;
    lds_barrier();
    if (any_hole(flags)) [[unlikely]] {
      for (int k0 = lo; k0 < hi; k0 += C::CAP) {
        if (k0 + C::CAP <= block_least) continue;
        lds_barrier();
        first = entry_of(a, x.slot, k0 + tid, hi);
        chunk(k0);
        for (int it = 0; it * KEYS < min(hi - k0, C::CAP); ++it) {
          if (k0 + (it + 1) * KEYS <= block_least) continue;
          places(it);
          dma(std::integral_constant<int, 0>{});
          landed<0>();
          lds_barrier();
          if (!idle)
            add_odd<DT, DP, NDB, KEYS / 16>(Ks + STAGES * TILE, lane, min(p.limit, hi) - k0 - it * KEYS,
                                            tok + it * KEYS, oacc);
          lds_barrier();
        }
      }
    }
  }
  const float l = run.l + __shfl_xor(run.l, 32, 64);
  if constexpr (ND > 192) {  // looked up again: its registers are the loop's
    const Pair e = pair_of(a, x, wave * 32 + (int)opaque(qi), alike);
    if (e.valid) store_partial<NDB>(a, e.part, oacc, run.m, l, hh);
  } else if (p.valid) {
    store_partial<NDB>(a, p.part, oacc, run.m, l, hh);
  }
}

// Up to 32 pairs: the four waves have the same pairs and take every fourth
// group of OWN keys each, through a K and a V tile of their own, with no barrier
// between them; their results are joined in LDS in a fixed order.  The next
// group's K is in flight from the scores on, its V from the product with V on.
// 16-key groups fill half of a 32-row score product; what a narrow item waits
// for is memory: 2 rows of 7 heads a kv head behind 128K tokens, D 64, 67 MB, 15
// us, 4.4 TB/s (a block of 128 pairs with 14 in use took 225).  SOLO: x is this
// wave's alone, and it takes every group: a short sequence's few keys are not
// worth a workgroup (225 sequences of up to 4 own tokens, 32 kv heads: 25 us, 58
// with a workgroup each), many are (64 of up to 2048: 174, 108).
template <int DT, int ND, bool NEAR, bool UNEVEN, bool SOLO>
MOBA_DEV void narrow_item(const SharedArgs& a, const Item& x, char* smem) {
  typedef Dims<ND> C;
  constexpr int DP = C::DP, NKS = C::NKS, NDB = C::NDB, NB = C::NB, OWN = C::OWN;
  constexpr int NDMA = OWN * NB / 64;  // loads of a K or V tile
  constexpr int NR = OWN / 2;          // score registers in use
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 31, hh = lane >> 5, D = a.D;
  uint16_t *Kt = (uint16_t*)smem + wave * 2 * OWN * DP, *Vt = Kt + OWN * DP;
  constexpr int CAP = SOLO ? C::CAP / 4 : C::CAP, STEP = SOLO ? 1 : 4;
  uint32_t* tok = (uint32_t*)(smem + C::TOK) + (SOLO ? wave * CAP : 0);
  int* flags = (int*)(smem + C::FLAGS);
  const int thread = SOLO ? lane : tid, begin = SOLO ? 0 : wave;

  const int alike = alike_of(a, x);
  int lo, hi, first = -1;
  range_of(x, alike, lo, hi);
  // what the keys wait for goes out first
  if (lo < hi) first = entry_of(a, x.slot, lo + thread, hi);
  const Pair p = pair_of(a, x, qi, alike);
  if (alike < 0) {
    range_of(x, longest(p.limit), lo, hi);
    if (lo < hi) first = entry_of(a, x.slot, lo + thread, hi);
  }
  if (lo >= hi) {
    if (thread < 32 && p.valid) a.part_ml[p.part] = make_float2(-INFINITY, 0.0f);
    return;
  }
  const Rows<NEAR> rows(a, x.kh);
  u16x8_t qf[NKS];
  load_query<NKS>(a, p, hh, qf);

  f32x16_t oacc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) oacc[db] = zero16();
  Running run;
  const int wlim = min(shortest(p, alike), hi);
  const uint32_t kbase0 = swz_b128_base<DP>(lane);
  const uint32_t trb0 = swz_tr_base<DP>(lane, 0), trb1 = swz_tr_base<DP>(lane, 1);
  const uint32_t lds0 = lds_addr(Kt);
  auto bring = [&](int it, auto v) {
    const uint32_t ln = opaque(lane);
#pragma unroll
    for (int n = 0; n < NDMA; ++n) {
      const uint32_t row0 = n * (64 / NB), byte = block_byte<DP>(ln, row0);
      const uint32_t at = tok[it * OWN + row0 + ln / NB];
      if (byte < (uint32_t)D * 2)
        rows.template bring<decltype(v)::value>(at, byte, lds0 + decltype(v)::value * (OWN * DP * 2) + n * 1024);
    }
  };
  auto chunk = [&](int k0) {
    bool holes = look_up<NEAR, CAP, SOLO ? 64 : 256>(a, rows, x.slot, k0, hi, first, thread, tok);
    if constexpr (SOLO) {
      wave_lds_sync();
    } else {
      if (lane == 0) flags[wave] = holes;
      lds_barrier();
      holes = any_hole(flags);
    }
    landed<0>();  // what the compiler has in flight: it must not wait for it below
    return holes;
  };
  bool odd = false;
  for (int k0 = lo; k0 < hi; k0 += CAP) {
    if (k0 > lo) {
      if constexpr (!SOLO) lds_barrier();  // the tokens before are read
      first = entry_of(a, x.slot, k0 + thread, hi);
    }
    const bool holes = chunk(k0);
    const int ntiles = (min(hi - k0, CAP) + OWN - 1) / OWN;
    if (begin < ntiles) {
      bring(begin, std::false_type{});
      bring(begin, std::true_type{});
    }
    for (int it = begin; it < ntiles; it += STEP) {
      const uint32_t kq = opaque(kbase0), t0 = opaque(trb0), t1 = opaque(trb1);
      const bool more = it + STEP < ntiles;
      landed<NDMA>();  // K; V may be on its way
      f32x16_t s[1] = {zero16()};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) s[0] = mfma32<DT>(lds8(Kt, swz_b128<DP>(kq, ks)), qf[ks], s[0]);
      lds_read_done();
      if (more) bring(it + STEP, std::false_type{});
      const int kt0 = k0 + it * OWN;
      const bool ends = UNEVEN && alike < 0 && kt0 + OWN > wlim;  // rows of unlike lengths
      if (kt0 + OWN > wlim || holes)
        mask_scores<1, NR>(s, min(p.limit, hi) - kt0, tok + it * OWN, hh);
      u16x8_t pv[1][NR / 8];
      softmax_step<DT, 1, NR, NDB>(s, a.scale_log2, run, oacc, pv);
      if (more) landed<NDMA>(); else landed<0>();  // V; the next K may be on its way
      if (ends) {
        odd |= odd_in<DT, OWN * DP, 64>(Vt, lane);
        wave_lds_sync();
      }
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int t = 0; t < NR / 8; ++t) {
          const uint32_t ro = t * 16 * DP * 2;
          oacc[db] = mfma32<DT>(lds_tr8(Vt, ro + swz_tr<DP>(t0, db), ro + swz_tr<DP>(t1, db)),
                                pv[0][t], oacc[db]);
        }
      lds_read_done();
      if (more) bring(it + STEP, std::true_type{});
    }
  }
  if (UNEVEN && alike < 0) {
    if constexpr (!SOLO) {
      lds_barrier();
      if (lane == 0) flags[wave] = odd;
      lds_barrier();
      odd = any_hole(flags);
    }
    if (odd) [[unlikely]]
      for (int k0 = lo; k0 < hi; k0 += CAP) {
        if (k0 + CAP <= wlim) continue;
        if constexpr (!SOLO) lds_barrier();
        first = entry_of(a, x.slot, k0 + thread, hi);
        chunk(k0);
        for (int it = begin; it * OWN < min(hi - k0, CAP); it += STEP) {
          if (k0 + (it + 1) * OWN <= wlim) continue;
          bring(it, std::true_type{});
          landed<0>();
          add_odd<DT, DP, NDB, OWN / 16>(Vt, lane, min(p.limit, hi) - k0 - it * OWN, tok + it * OWN, oacc);
          lds_read_done();
        }
      }
  }
  float m_run = run.m, l = run.l + __shfl_xor(run.l, 32, 64);
  if constexpr (SOLO) {
    if (p.valid) store_partial<NDB>(a, p.part, oacc, m_run, l, hh);
    return;
  }

  // Join, lane by lane, waves in order: wave w takes the 32-dim blocks db % 4 ==
  // w from the others and writes them, four blocks a round.
  f32x4_t* ox = (f32x4_t*)smem;                // [4 waves][3][4][64], where the tiles were
  float2* mx = (float2*)(smem + C::TOK);       // [4][64]
  lds_barrier();                               // tiles and tokens are read
  mx[wave * 64 + lane] = make_float2(m_run, l);
  float weight[4];
  float* po = a.part_o + p.part * D;
#pragma unroll
  for (int b0 = 0; b0 < NDB; b0 += 4) {
    if (b0) lds_barrier();                     // the round before is read
#pragma unroll
    for (int i = 0; i < 4 && b0 + i < NDB; ++i)
      if (i != wave) {
        const int at = (wave * 3 + (i > wave ? i - 1 : i)) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          ox[(at + j) * 64 + lane] = (f32x4_t){oacc[b0 + i][4 * j], oacc[b0 + i][4 * j + 1],
                                               oacc[b0 + i][4 * j + 2], oacc[b0 + i][4 * j + 3]};
      }
    lds_barrier();
    if (b0 == 0) {
      float2 ml[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) ml[w] = mx[w * 64 + lane];
      m_run = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
      const float ref = m_run == -INFINITY ? 0.0f : m_run;
      l = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        weight[w] = fast_exp2(ml[w].x - ref);
        l += ml[w].y * weight[w];
      }
      if (wave == 0 && p.valid && hh == 0) a.part_ml[p.part] = make_float2(m_run, l);
    }
#pragma unroll
    for (int i = 0; i < 4 && b0 + i < NDB; ++i)
      if (i == wave) {
        f32x4_t sum[4];
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f32x4_t v = {oacc[b0 + i][4 * j], oacc[b0 + i][4 * j + 1], oacc[b0 + i][4 * j + 2],
                         oacc[b0 + i][4 * j + 3]};
            if (w != i) v = ox[((w * 3 + (i > w ? i - 1 : i)) * 4 + j) * 64 + lane];
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[j][k] = w ? fmaf(v[k], weight[w], sum[j][k]) : v[k] * weight[0];
          }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = (b0 + i) * 32 + 8 * j + 4 * hh;
          if (p.valid && d < D) *reinterpret_cast<f32x4_t*>(po + d) = sum[j];
        }
      }
  }
}

template <int DT, int ND, bool NEAR, bool UNEVEN>
__global__ __launch_bounds__(256, Dims<ND>::WAVES) void block_kernel(SharedArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[Dims<ND>::LDS];
  const Item x = a.items[blockIdx.x];
  if (x.n_m == 0) return;
  // Dims behind D are never loaded: zeros where they are multiplied, or looked at
  if (a.D < ND || (UNEVEN && a.D < Dims<ND>::DP && x.length < 0)) {
    for (int i = threadIdx.x * 16; i < Dims<ND>::TILES; i += 4096) st8((uint16_t*)(smem + i), zero8());
    lds_barrier();
  }
  if (x.n_m < 0) {
    const Item own = a.items[x.row_at + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)];
    if (own.n_m > 0) narrow_item<DT, ND, NEAR, UNEVEN, true>(a, own, smem);
  } else if (x.n_m <= 32) narrow_item<DT, ND, NEAR, UNEVEN, false>(a, x, smem);
  else wide_item<DT, ND, NEAR, UNEVEN>(a, x, smem);
}

// Joins the ranges of each (row, head): PL threads per four dims, each with
// every PL-th range, four of them at a time (their loads are in flight
// together), then the PL sums in LDS in order.  Bound by the reads of the
// partials: 5 ranges of 16384 (row, head)s of 256 dims, 84 MB, 16.8 us, 5.0 TB/s
// (they come from the last-level cache); with few rows by the latency of the two
// dependent loads, 3 to 5 us.
template <int DT>
__global__ __launch_bounds__(256) void merge_kernel(const float* __restrict__ part_o,
                                                    const float2* __restrict__ part_ml,
                                                    const int* __restrict__ part_at,
                                                    const int* __restrict__ n_part, int n_rows,
                                                    int Hq, int D, int PL,
                                                    uint16_t* __restrict__ out,
                                                    float* __restrict__ lse) {
  __shared__ f32x4_t red[256];
  __shared__ float2 ml_red[256];
  const int tpr = D / 4, tpp = tpr * PL, per = 256 / tpp;
  const int e = threadIdx.x / tpp, in = threadIdx.x - e * tpp, pl = in / tpr;
  const int d = (in - pl * tpr) * 4;
  const int64_t rh = (int64_t)blockIdx.x * per + e;
  const bool on = e < per && rh < (int64_t)n_rows * Hq;
  const int row = on ? (int)(rh / Hq) : 0, h = on ? (int)(rh - (int64_t)row * Hq) : 0;
  const int n = on ? n_part[row] : 0;
  const int64_t s0 = (int64_t)part_at[row] * Hq + h;
  float M = -INFINITY, z = 0.0f;
  f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = pl; i0 < n; i0 += 4 * PL) {
    float2 ml[4];
    f32x4_t v[4];
    float mn = M;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * PL;
      const int64_t s = s0 + (int64_t)min(i, n - 1) * Hq;
      ml[k] = part_ml[s];
      v[k] = *reinterpret_cast<const f32x4_t*>(part_o + s * D + d);
      if (i >= n) ml[k].y = 0.0f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (ml[k].y != 0.0f) mn = fmaxf(mn, ml[k].x);
    const float keep = M == -INFINITY ? 0.0f : fast_exp2(M - mn);
    M = mn;
    z *= keep;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] *= keep;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool some = ml[k].y != 0.0f;  // an empty range wrote no O
      const float w = some ? fast_exp2(ml[k].x - mn) : 0.0f;
      z += some ? w * ml[k].y : 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] += some ? w * v[k][c] : 0.0f;
    }
  }
  if (PL > 1) {
    ml_red[threadIdx.x] = make_float2(M, z);
    red[threadIdx.x] = o;
    __syncthreads();
    if (pl != 0 || !on) return;
    float top = M;
    for (int k = 1; k < PL; ++k) top = fmaxf(top, ml_red[threadIdx.x + k * tpr].x);
    const float ref = top == -INFINITY ? 0.0f : top, w0 = fast_exp2(M - ref);
    M = top;
    z *= w0;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] *= w0;
    for (int k = 1; k < PL; ++k) {
      const float2 ml = ml_red[threadIdx.x + k * tpr];
      const f32x4_t v = red[threadIdx.x + k * tpr];
      const float w = fast_exp2(ml.x - ref);
      z += w * ml.y;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] += w * v[c];
    }
  }
  if (!on) return;
  const float inv = z != 0.0f ? 1.0f / z : 0.0f;
  uint2 w2;
  w2.x = pack2<DT>(o[0] * inv, o[1] * inv);
  w2.y = pack2<DT>(o[2] * inv, o[3] * inv);
  *reinterpret_cast<uint2*>(out + rh * D + d) = w2;
  if (d == 0) lse[rh] = z != 0.0f ? (M + log2f(z)) * kLn2 : -INFINITY;
}

template <int DT, bool NEAR, bool UNEVEN> void launch_blocks(const SharedArgs& a, int n_items, hipStream_t st) {
  const dim3 grid(n_items), block(256);
  if (a.D <= 64) hipLaunchKernelGGL((block_kernel<DT, 64, NEAR, UNEVEN>), grid, block, 0, st, a);
  else if (a.D <= 96) hipLaunchKernelGGL((block_kernel<DT, 96, NEAR, UNEVEN>), grid, block, 0, st, a);
  else if (a.D <= 128) hipLaunchKernelGGL((block_kernel<DT, 128, NEAR, UNEVEN>), grid, block, 0, st, a);
  else if (a.D <= 192) hipLaunchKernelGGL((block_kernel<DT, 192, NEAR, UNEVEN>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((block_kernel<DT, 256, NEAR, UNEVEN>), grid, block, 0, st, a);
}

template <int DT>
void launch_merge(const SharedArgs& a, int Nq, int max_parts, uint16_t* out, float* lse,
                  hipStream_t st) {
  // A thread takes the ranges four at a time.  One round of them is fastest
  // while the launch is small (us with 1, 4, 16 threads per dims: 154 ranges of 28
  // (row, head) pairs 23.6, 8.5, 5.0; 17 of 1512 5.1, 4.4, 5.9); one that fills
  // the card by itself has its loads in flight anyway (11 of 8192: 10.8, 14.2).
  int pl = 1;
  const int64_t threads = (int64_t)Nq * a.Hq * (a.D / 4);
  while (4 * pl < max_parts && pl * threads < 65536 && 2 * pl * (a.D / 4) <= 256) pl *= 2;
  const int per = 256 / (a.D / 4 * pl);
  const dim3 grid((unsigned)(((int64_t)Nq * a.Hq + per - 1) / per));
  hipLaunchKernelGGL((merge_kernel<DT>), grid, dim3(256), 0, st, a.part_o, a.part_ml, a.prefix_at,
                     a.n_part, Nq, a.Hq, a.D, pl, out, lse);
}

}  // namespace

extern "C" int moba_hip_shared_attention(const void* q, int dtype, int Nq, int Hq, int Hkv, int D,
                                         float scale, const void* k_cache, const void* v_cache,
                                         int num_pages, int page_size, const int* table,
                                         int table_width, const int* own_lengths, int length_add, int max_length,
                                         const int* items, int n_items, const int* rows,
                                         const int* row_parts, int max_parts, int uneven, float* part_o, float* part_ml,
                                         void* out, float* lse, void* stream) {
  if (dtype != 0 && dtype != 1) { moba_set_error("shared_attention: dtype must be 0 (bf16) or 1 (fp16)"); return MOBA_ERR_ARG; }
  if (D < 8 || D > 256 || D % 8) { moba_set_error("shared_attention: head_dim must be a multiple of 8 in [8,256]"); return MOBA_ERR_ARG; }
  if (Nq < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || (int64_t)Nq * Hq >= 1ll << 31) { moba_set_error("shared_attention: Nq * Hq in [1, 2^31) and Hq a multiple of Hkv required"); return MOBA_ERR_ARG; }
  if (!(scale >= 0x1p-126f) || scale > 1e30f) { moba_set_error("shared_attention: scale must be positive and finite, in [2^-126, 1e30]"); return MOBA_ERR_ARG; }
  if (num_pages < 1 || page_size < 1 || table_width < 1 || (int64_t)num_pages * page_size >= 1ll << 31 ||
      (int64_t)table_width * page_size >= 1ll << 31) { moba_set_error("shared_attention: nonempty page pool and table below 2^31 tokens required"); return MOBA_ERR_ARG; }
  if ((int64_t)Hkv * D >= 1ll << 30) { moba_set_error("shared_attention: Hkv * D below 2^30 required"); return MOBA_ERR_ARG; }
  // (at most 2^30: a group of keys behind the last still counts in 32 bits)
  if (n_items < 0 || max_length < 0 || max_length > table_width * page_size || max_length > 1 << 30) { moba_set_error("shared_attention: max_length must be at most 2^30 and fit the page table"); return MOBA_ERR_ARG; }
  SharedArgs a;
  a.q = (const uint16_t*)q; a.kc = (const uint16_t*)k_cache; a.vc = (const uint16_t*)v_cache;
  a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.G = Hq / Hkv;
  a.scale_log2 = scale * kLog2e;
  a.num_pages = num_pages; a.P = page_size; a.W = table_width; a.table = table;
  a.lengths = own_lengths; a.length_add = length_add; a.max_length = max_length;
  a.items = (const Item*)items; a.rows = rows;
  const int64_t pool = (int64_t)num_pages * page_size * Hkv * D * 2;
  a.pool_bytes = pool <= kNowhere ? (uint32_t)pool : 0;
  a.prefix_at = row_parts; a.own_at = row_parts + Nq; a.n_part = row_parts + 2 * (int64_t)Nq;
  a.part_o = part_o; a.part_ml = (float2*)part_ml;
  hipStream_t st = (hipStream_t)stream;
  if (n_items > 0) {
    // Pools above 4 GiB have the one kernel for all plans (64 rows behind 32K tokens 110
    // us a call there and below; 256 rows 198, 185 below; 8 behind 2K 11.4, 11.2)
    if (!a.pool_bytes) dtype == 0 ? launch_blocks<0, false, true>(a, n_items, st) : launch_blocks<1, false, true>(a, n_items, st);
    else if (uneven) dtype == 0 ? launch_blocks<0, true, true>(a, n_items, st) : launch_blocks<1, true, true>(a, n_items, st);
    else dtype == 0 ? launch_blocks<0, true, false>(a, n_items, st) : launch_blocks<1, true, false>(a, n_items, st);
    const int rc = moba_launch_status("shared_attention(blocks)");
    if (rc) return rc;
  }
  if (dtype == 0) launch_merge<0>(a, Nq, max_parts, (uint16_t*)out, lse, st);
  else launch_merge<1>(a, Nq, max_parts, (uint16_t*)out, lse, st);
  return moba_launch_status("shared_attention(merge)");
}
