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
#include "common.h"
#include "../../include/moba_hip.h"

using namespace moba;

namespace {

// One work item (the plan's int32 record).
struct Item {
  int row_at;   // its segment's first entry of `rows`
  int m0;       // first (row, q head of the kv head) pair of the block: row m / G
  int n_m;      // pairs of the block
  int slot;     // page-table row of the keys
  int kh;
  int split, splits;
  int length;   // tokens of the segment; -1: each row's own length
};

struct SharedArgs {
  const uint16_t *q, *kc, *vc;
  int Hq, Hkv, D, G;
  float scale_log2;
  int num_pages, P, W;
  const int* table;
  const int* lengths;       // own tokens of each row
  int max_length;
  const Item* items;
  const int* rows;
  const int *part_at, *n_prefix, *n_part;  // per row: first partial, prefix ranges, ranges
  float* part_o;
  float2* part_ml;
};

constexpr uint32_t kNoToken = 0xffffffffu;

// What a key of no token loads: zeros, so that a weight of 0 meets no NaN.
__device__ __attribute__((aligned(16))) const uint16_t g_zero[8] = {0};

// 16 bytes per lane from any address straight into LDS (lane l's at
// lds + 16 l); ordered by the caller as dma_lds16.
MOBA_DEV void dma_global16(const void* p, const void* lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds_addr(lds)), "v"(p) : "memory", "m0");
}

// Sizes of a head dim's kernel.
template <int ND> struct Dims {
  static constexpr int DP = ND <= 64 ? 64 : ND <= 128 ? 128 : 256;  // row of the LDS layouts
  static constexpr int NKS = ND / 16, NDB = ND / 32, NB = DP / 8;
  static constexpr int KEYS = DP <= 64 ? 64 : 32;  // keys of a tile that four waves share
  static constexpr int TILE = KEYS * DP;
  // bytes of LDS: two stages of K and V tiles, looked-up tokens and flags; or a
  // V tile per wave and the query rows
  static constexpr int TOK = 4 * TILE * 2, FLAGS = TOK + 2 * 256 * 4, WIDE = FLAGS + 8 * 4;
  static constexpr int ROWS = 4 * 32 * DP * 2, NARROW = ROWS + 32 * DP * 2;
  static constexpr int LDS = WIDE > NARROW ? WIDE : NARROW;
  static constexpr int WAVES = ND <= 128 ? 3 : 2;  // per SIMD
};

// What a lane knows of its (row, q head) pair.
struct Pair {
  int row, h, limit;
  bool valid;
};
MOBA_DEV Pair pair_of(const SharedArgs& a, const Item& x, int m) {
  Pair p;
  p.valid = m < x.n_m;
  const int i = x.m0 + min(m, x.n_m - 1);
  p.row = a.rows[x.row_at + i / a.G];
  p.h = x.kh * a.G + i % a.G;
  p.limit = x.length < 0 ? max(0, min(a.lengths[p.row], a.max_length)) : x.length;
  return p;
}
MOBA_DEV int64_t partial_of(const SharedArgs& a, const Item& x, const Pair& p) {
  return ((int64_t)a.part_at[p.row] + (x.length < 0 ? a.n_prefix[p.row] : 0) + x.split) * a.Hq + p.h;
}
// The keys [lo, hi) of an item's range: whole groups of 64 but for the last.
MOBA_DEV void range_of(const Item& x, int length, int& lo, int& hi) {
  const int per = ((length + 64 * x.splits - 1) / (64 * x.splits)) * 64;
  lo = min(length, x.split * per);
  hi = min(length, lo + per);
}
// The pool's token of key `key` of a slot.
MOBA_DEV uint32_t token_of(const SharedArgs& a, const int* trow, int key, int hi) {
  const int k = min(key, hi - 1), lp = k / a.P, page = trow[lp];
  const bool on = key < hi && page >= 0 && page < a.num_pages;
  return on ? (uint32_t)page * a.P + (k - lp * a.P) : kNoToken;
}

template <int NDB>
MOBA_DEV void store_partial(const SharedArgs& a, int64_t slot, const f32x16_t (&o)[NDB], float m,
                            float l, int hh) {
  float* po = a.part_o + slot * a.D;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = db * 32 + 8 * j + 4 * hh;
      if (d < a.D)
        *reinterpret_cast<f32x4_t*>(po + d) =
            (f32x4_t){o[db][4 * j], o[db][4 * j + 1], o[db][4 * j + 2], o[db][4 * j + 3]};
    }
  if (hh == 0) a.part_ml[slot] = make_float2(m, l);
}

// One tile's scores into the running (max, sum) of a lane's pair; returns the
// 16-bit weights as operands of the product with V.
template <int DT, int NKB, int NDB>
MOBA_DEV void softmax_step(const f32x16_t (&s)[NKB], float c2, float& m_run, float& lsum,
                           f32x16_t (&o)[NDB], u16x8_t (&pv)[NKB][2]) {
  float mx = -INFINITY;
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
  mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c2;
  const bool up = mx > m_run;
  if (__any(up)) {
    const float mn = up ? mx : m_run;
    const float alpha = up ? fast_exp2(m_run - mn) : 1.0f;
    lsum *= alpha;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
    m_run = mn;
  }
  // a row with nothing so far: weights of 0, not of exp2(-inf + inf)
  const float nm = m_run == -INFINITY ? 0.0f : -m_run;
  float ps = 0.0f;
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb) {
    float p[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] = fast_exp2(fmaf(s[kb][r], c2, nm));
      ps += p[r];
    }
    pv[kb][0] = pack8<DT>(p);
    pv[kb][1] = pack8<DT>(p + 8);
  }
  lsum += ps;
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

// More than 32 pairs: every wave has 32 of them, and the four share tiles of
// KEYS keys in two LDS stages.
template <int DT, int ND>
MOBA_DEV void wide_item(const SharedArgs& a, const Item& x, char* smem) {
  typedef Dims<ND> C;
  uint32_t (*tok)[256] = (uint32_t(*)[256])(smem + C::TOK);  // pool token of each key
  int* flags = (int*)(smem + C::FLAGS);
  constexpr int DP = C::DP, NKS = C::NKS, NDB = C::NDB, KEYS = C::KEYS, NKB = KEYS / 32;
  constexpr int TILE = C::TILE, NB = C::NB, NDMA = KEYS * NB / 256;
  constexpr int TPC = 256 / KEYS;   // tiles per 256 looked-up tokens
  uint16_t* Ks = (uint16_t*)smem;   // [2][TILE], then V
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 31, hh = lane >> 5, D = a.D;

  const Pair p = pair_of(a, x, wave * 32 + qi);
  int length = x.length;
  if (length < 0) {  // the block's longest row
    int mx = p.limit;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = max(mx, __shfl_xor(mx, o, 64));
    if (lane == 0) flags[wave] = mx;
    lds_barrier();
    length = max(max(flags[0], flags[1]), max(flags[2], flags[3]));
    lds_barrier();
  }
  int lo, hi;
  range_of(x, length, lo, hi);
  if (lo >= hi) {
    if (p.valid && hh == 0) a.part_ml[partial_of(a, x, p)] = make_float2(-INFINITY, 0.0f);
    return;
  }

  const int* trow = a.table + (int64_t)x.slot * a.W;
  auto publish = [&](int c, uint32_t t) {  // this thread's key of chunk c of 256
    tok[c & 1][tid] = t;
    const bool any = __any(t == kNoToken);
    if (lane == 0) flags[4 * (c & 1) + wave] = any;
  };
  const char *kp = (const char*)(a.kc + (int64_t)x.kh * D), *vp = (const char*)(a.vc + (int64_t)x.kh * D);
  const uint32_t row_bytes = (uint32_t)(a.Hkv * D * 2);
  // thread (wave w, lane l) brings 16-byte blocks j = (n * 4 + w) * 64 + l of a
  // tile: row j / NB, physical block j % NB of the swizzled row
  auto dma = [&](int it) {
    const uint32_t* tk = &tok[(it / TPC) & 1][(it % TPC) * KEYS];
    uint16_t* Kd = Ks + (it & 1) * TILE;
    const uint32_t ln = opaque(lane);
#pragma unroll
    for (int n = 0; n < NDMA; ++n) {
      const uint32_t row0 = (n * 4 + wave) * (64 / NB), byte = block_byte<DP>(ln, row0);
      if (byte < ND * 2) {
        const uint32_t t = tk[row0 + ln / NB];
        const bool on = (t != kNoToken) & (byte < (uint32_t)D * 2);
        const uint64_t off = (uint64_t)t * row_bytes + byte;
        dma_global16(on ? kp + off : (const char*)g_zero, Kd + (n * 4 + wave) * 64 * 8);
        dma_global16(on ? vp + off : (const char*)g_zero, Kd + 2 * TILE + (n * 4 + wave) * 64 * 8);
      }
    }
  };

  publish(0, token_of(a, trow, lo + tid, hi));
  u16x8_t qf[NKS];
  const uint16_t* qrow = a.q + ((int64_t)p.row * a.Hq + p.h) * D;
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) {
    const int d = ks * 16 + hh * 8;
    const u16x8_t v = ld8(qrow + (d < D ? d : 0));
    qf[ks] = d < D ? v : zero8();
  }
  lds_barrier();
  dma(0);

  f32x16_t oacc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) oacc[db] = zero16();
  float m_run = -INFINITY, lsum = 0.0f;
  const bool idle = wave * 32 >= x.n_m;
  int wlim = p.valid ? p.limit : 0x7fffffff;  // the wave's shortest row
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wlim = min(wlim, __shfl_xor(wlim, o, 64));
  wlim = __builtin_amdgcn_readfirstlane(wlim);

  const uint32_t kbase0 = swz_b128_base<DP>(lane);
  const uint32_t trb0 = swz_tr_base<DP>(lane, 0), trb1 = swz_tr_base<DP>(lane, 1);
  auto tile = [&](int it) {
    const uint16_t *Kb = Ks + (it & 1) * TILE, *Vb = Kb + 2 * TILE;
    const uint32_t kq = opaque(kbase0), t0 = opaque(trb0), t1 = opaque(trb1);
    const int kt0 = lo + it * KEYS;
    f32x16_t sacc[NKB];
    wave_prio<1>();
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
      sacc[kb] = zero16();
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
        sacc[kb] = mfma32<DT>(lds8(Kb, kb * 32 * DP * 2 + swz_b128<DP>(kq, ks)), qf[ks], sacc[kb]);
    }
    wave_prio<0>();
    const int at = (it % TPC) * KEYS, c = (it / TPC) & 1;
    if (kt0 + KEYS > wlim || __builtin_amdgcn_readfirstlane(flags[4 * c + at / 64])) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int k = kb * 32 + 8 * j + 4 * hh;
          const u32x4_t t = *reinterpret_cast<const u32x4_t*>(&tok[c][at + k]);
          const int left = (int)opaque(p.limit - kt0) - k;  // keys from k on below the limit
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sacc[kb][4 * j + i] = (i < left) & (t[i] != kNoToken) ? sacc[kb][4 * j + i] : -INFINITY;
        }
    }
    u16x8_t pv[NKB][2];
    softmax_step<DT, NKB, NDB>(sacc, a.scale_log2, m_run, lsum, oacc, pv);
    wave_prio<1>();
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t ro = (kb * 32 + t * 16) * DP * 2;
          oacc[db] = mfma32<DT>(lds_tr8(Vb, ro + swz_tr<DP>(t0, db), ro + swz_tr<DP>(t1, db)),
                                pv[kb][t], oacc[db]);
        }
    wave_prio<0>();
  };

  const int ntiles = (hi - lo + KEYS - 1) / KEYS;
  for (int it = 0; it < ntiles; ++it) {
    wait_vmcnt<0>();  // this wave's part of tile `it` has landed
    lds_barrier();    // everyone's has, and tile it - 1 is read
    uint32_t next = 0;
    const bool more = it % TPC == 0 && (it / TPC + 1) * TPC < ntiles;
    if (more) next = token_of(a, trow, lo + (it / TPC + 1) * 256 + tid, hi);
    if (it + 1 < ntiles) dma(it + 1);
    if (!idle) tile(it);
    if (more) publish(it / TPC + 1, next);  // read from tile it + TPC - 1 on
  }
  const float l = lsum + __shfl_xor(lsum, 32, 64);
  if (p.valid) store_partial<NDB>(a, partial_of(a, x, p), oacc, m_run, l, hh);
}

// Up to 32 pairs: the four waves have the same pairs and take every fourth
// group of 32 keys each, the K rows straight into registers, the V rows into
// an LDS tile of their own, with no barrier between them; their results are
// joined in LDS in a fixed order.
template <int DT, int ND>
MOBA_DEV void narrow_item(const SharedArgs& a, const Item& x, char* smem) {
  typedef Dims<ND> C;
  constexpr int DP = C::DP, NKS = C::NKS, NDB = C::NDB, NB = C::NB;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 31, hh = lane >> 5, D = a.D;
  uint16_t* Vs = (uint16_t*)smem + wave * 32 * DP;
  uint16_t* Qs = (uint16_t*)(smem + C::ROWS);

  const Pair p = pair_of(a, x, qi);
  int length = p.limit;  // the longest row (static: everyone's)
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) length = max(length, __shfl_xor(length, o, 64));
  length = __builtin_amdgcn_readfirstlane(length);
  int lo, hi;
  range_of(x, length, lo, hi);
  if (lo >= hi) {
    if (tid < 32 && p.valid) a.part_ml[partial_of(a, x, p)] = make_float2(-INFINITY, 0.0f);
    return;
  }

  const int* trow = a.table + (int64_t)x.slot * a.W;
  const char *kp = (const char*)(a.kc + (int64_t)x.kh * D), *vp = (const char*)(a.vc + (int64_t)x.kh * D);
  const uint32_t row_bytes = (uint32_t)(a.Hkv * D * 2);
  const int ntiles = (hi - lo + 31) / 32;
  u16x8_t kf[NKS];
  auto load_k = [&](uint32_t t) {
    // a key of no token loads the pool's first one: its score is masked
    const uint16_t* row = (const uint16_t*)(kp + (uint64_t)(t != kNoToken ? t : 0) * row_bytes);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) {
      const int d = ks * 16 + hh * 8;
      const u16x8_t v = ld8(row + (d < D ? d : 0));
      kf[ks] = d < D ? v : zero8();
    }
  };
  auto load_v = [&](uint32_t t) {
    const uint32_t ln = opaque(lane);
#pragma unroll
    for (int n = 0; n < NB / 2; ++n) {
      const uint32_t row0 = n * (64 / NB), byte = block_byte<DP>(ln, row0);
      const uint32_t tr = __shfl(t, row0 + ln / NB, 64);
      if (byte < ND * 2) {
        const bool on = (tr != kNoToken) & (byte < (uint32_t)D * 2);
        dma_global16(on ? vp + ((uint64_t)tr * row_bytes + byte) : (const char*)g_zero, Vs + n * 64 * 8);
      }
    }
  };
  uint32_t t_now = token_of(a, trow, lo + wave * 32 + qi, hi), t_next = kNoToken;
  if (wave < ntiles) {
    load_k(t_now);
    load_v(t_now);
    t_next = token_of(a, trow, lo + (wave + 4) * 32 + qi, hi);
  }
  // the query rows, once for the four waves
  const uint16_t* qrow = a.q + ((int64_t)p.row * a.Hq + p.h) * D;
  const uint32_t kbase0 = swz_b128_base<DP>(lane);
  for (int ks = wave; ks < NKS; ks += 4) {
    const int d = ks * 16 + hh * 8;
    const u16x8_t v = ld8(qrow + (d < D ? d : 0));
    st8((uint16_t*)((char*)Qs + swz_b128<DP>(kbase0, ks)), d < D ? v : zero8());
  }
  int wlim = p.valid ? p.limit : 0x7fffffff;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wlim = min(wlim, __shfl_xor(wlim, o, 64));
  wlim = __builtin_amdgcn_readfirstlane(wlim);
  lds_barrier();

  f32x16_t oacc[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) oacc[db] = zero16();
  float m_run = -INFINITY, lsum = 0.0f;
  const uint32_t trb0 = swz_tr_base<DP>(lane, 0), trb1 = swz_tr_base<DP>(lane, 1);
  for (int it = wave; it < ntiles; it += 4) {
    f32x16_t s[1] = {zero16()};
    const uint32_t kq = opaque(kbase0), t0 = opaque(trb0), t1 = opaque(trb1);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) s[0] = mfma32<DT>(kf[ks], lds8(Qs, swz_b128<DP>(kq, ks)), s[0]);
    const uint32_t live = (uint32_t)__ballot(t_now != kNoToken);
    wait_vmcnt<0>();  // the V rows of this group have landed
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);  // the next K rows take the registers of these
    const bool more = it + 4 < ntiles;
    if (more) {
      t_now = t_next;
      load_k(t_now);
      t_next = token_of(a, trow, lo + (it + 8) * 32 + qi, hi);
    }
    const int kt0 = lo + it * 32;
    if (kt0 + 32 > wlim || live != 0xffffffffu) {
      const int left = (int)opaque(p.limit - kt0) - 4 * hh;
      const uint32_t mine = live >> (4 * hh);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int k = 8 * (r >> 2) + (r & 3);
        s[0][r] = (k < left) & ((mine >> k) & 1) ? s[0][r] : -INFINITY;
      }
    }
    u16x8_t pv[1][2];
    softmax_step<DT, 1, NDB>(s, a.scale_log2, m_run, lsum, oacc, pv);
    asm volatile("" ::: "memory");
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t ro = t * 16 * DP * 2;
        oacc[db] = mfma32<DT>(lds_tr8(Vs, ro + swz_tr<DP>(t0, db), ro + swz_tr<DP>(t1, db)),
                              pv[0][t], oacc[db]);
      }
    if (more) {
      __builtin_amdgcn_s_waitcnt(0xC07F);  // the V tile is read
      asm volatile("" ::: "memory");
      load_v(t_now);
    }
  }
  float l = lsum + __shfl_xor(lsum, 32, 64);

  // join: waves 2, 3 into 0, 1, then 1 into 0; lane by lane
  f32x4_t* ox = (f32x4_t*)smem;                        // [2][NDB * 4][64]
  float2* mx = (float2*)(smem + C::ROWS);      // [2][64], where the queries were
#pragma unroll
  for (int step = 2; step > 0; step >>= 1) {
    lds_barrier();
    const bool give = wave >= step && wave < 2 * step;
    const int at = give ? wave - step : wave;
    if (give) {
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          ox[(at * NDB * 4 + db * 4 + j) * 64 + lane] =
              (f32x4_t){oacc[db][4 * j], oacc[db][4 * j + 1], oacc[db][4 * j + 2], oacc[db][4 * j + 3]};
      mx[at * 64 + lane] = make_float2(m_run, l);
    }
    lds_barrier();
    if (wave < step) {
      const float2 o = mx[at * 64 + lane];
      const float M = fmaxf(m_run, o.x), ref = M == -INFINITY ? 0.0f : M;
      const float wa = fast_exp2(m_run - ref), wb = fast_exp2(o.x - ref);
      l = l * wa + o.y * wb;
      m_run = M;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4_t v = ox[(at * NDB * 4 + db * 4 + j) * 64 + lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) oacc[db][4 * j + i] = oacc[db][4 * j + i] * wa + v[i] * wb;
          __builtin_amdgcn_sched_barrier(0);  // 16 values at a time, not all in registers
        }
    }
  }
  if (wave == 0 && p.valid) store_partial<NDB>(a, partial_of(a, x, p), oacc, m_run, l, hh);
}

template <int DT, int ND>
__global__ __launch_bounds__(256, Dims<ND>::WAVES) void block_kernel(SharedArgs a) {
  __shared__ __attribute__((aligned(16))) char smem[Dims<ND>::LDS];
  const Item x = a.items[blockIdx.x];
  if (x.n_m == 0) return;
  if (x.n_m <= 32) narrow_item<DT, ND>(a, x, smem);
  else wide_item<DT, ND>(a, x, smem);
}

// Joins the ranges of each (row, head): a workgroup per pair (or several, PL
// = 1), PL threads per four dims, each with every PL-th range.
template <int DT, int PL>
__global__ __launch_bounds__(256) void merge_kernel(const float* __restrict__ part_o,
                                                    const float2* __restrict__ part_ml,
                                                    const int* __restrict__ part_at,
                                                    const int* __restrict__ n_part, int n_rows,
                                                    int Hq, int D, uint16_t* __restrict__ out,
                                                    float* __restrict__ lse) {
  __shared__ f32x4_t red[PL > 1 ? 256 : 1];
  __shared__ float2 ml_red[PL > 1 ? 256 : 1];
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
  // four ranges at a time: their loads are in flight together
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
      if (ml[k].y != 0.0f) mn = fmaxf(mn, ml[k].x);
    }
    const float keep = M == -INFINITY ? 0.0f : fast_exp2(M - mn);
    M = mn;
    z *= keep;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] *= keep;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (ml[k].y == 0.0f) continue;  // an empty range wrote no O
      const float w = fast_exp2(ml[k].x - mn);
      z += w * ml[k].y;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] += w * v[k][c];
    }
  }
  if constexpr (PL > 1) {
    ml_red[threadIdx.x] = make_float2(M, z);
    red[threadIdx.x] = o;
    __syncthreads();
    if (pl != 0) return;
    float Mx = M;
#pragma unroll
    for (int k = 1; k < PL; ++k) Mx = fmaxf(Mx, ml_red[threadIdx.x + k * tpr].x);
    const float ref = Mx == -INFINITY ? 0.0f : Mx;
    const float w0 = fast_exp2(M - ref);
    M = Mx;
    z *= w0;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] *= w0;
#pragma unroll
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

template <int DT> void launch_blocks(const SharedArgs& a, int n_items, hipStream_t st) {
  const dim3 grid(n_items), block(256);
  if (a.D <= 64) hipLaunchKernelGGL((block_kernel<DT, 64>), grid, block, 0, st, a);
  else if (a.D <= 96) hipLaunchKernelGGL((block_kernel<DT, 96>), grid, block, 0, st, a);
  else if (a.D <= 128) hipLaunchKernelGGL((block_kernel<DT, 128>), grid, block, 0, st, a);
  else if (a.D <= 192) hipLaunchKernelGGL((block_kernel<DT, 192>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((block_kernel<DT, 256>), grid, block, 0, st, a);
}

template <int DT, int PL>
void launch_merge(const SharedArgs& a, int Nq, uint16_t* out, float* lse, hipStream_t st) {
  const int per = 256 / (a.D / 4 * PL);
  const dim3 grid((unsigned)(((int64_t)Nq * a.Hq + per - 1) / per));
  hipLaunchKernelGGL((merge_kernel<DT, PL>), grid, dim3(256), 0, st, a.part_o, a.part_ml, a.part_at,
                     a.n_part, Nq, a.Hq, a.D, out, lse);
}

}  // namespace

extern "C" int moba_hip_shared_attention(const void* q, int dtype, int Nq, int Hq, int Hkv, int D,
                                         float scale, const void* k_cache, const void* v_cache,
                                         int num_pages, int page_size, const int* table,
                                         int table_width, const int* own_lengths, int max_length,
                                         const int* items, int n_items, const int* rows,
                                         const int* row_parts, int max_parts, float* part_o, float* part_ml,
                                         void* out, float* lse, void* stream) {
  if (dtype != 0 && dtype != 1) { moba_set_error("shared_attention: dtype must be 0 (bf16) or 1 (fp16)"); return MOBA_ERR_ARG; }
  if (D < 8 || D > 256 || D % 8) { moba_set_error("shared_attention: head_dim must be a multiple of 8 in [8,256]"); return MOBA_ERR_ARG; }
  if (Nq < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || (int64_t)Nq * Hq >= 1ll << 31) { moba_set_error("shared_attention: Nq * Hq in [1, 2^31) and Hq a multiple of Hkv required"); return MOBA_ERR_ARG; }
  if (!(scale > 0.0f) || scale > 1e30f) { moba_set_error("shared_attention: scale must be positive and finite"); return MOBA_ERR_ARG; }
  if (num_pages < 1 || page_size < 1 || table_width < 1 || (int64_t)num_pages * page_size >= 1ll << 31 ||
      (int64_t)table_width * page_size >= 1ll << 31) { moba_set_error("shared_attention: nonempty page pool and table below 2^31 tokens required"); return MOBA_ERR_ARG; }
  if (n_items < 0 || max_length < 0 || max_length > table_width * page_size) { moba_set_error("shared_attention: max_length must fit the page table"); return MOBA_ERR_ARG; }
  SharedArgs a;
  a.q = (const uint16_t*)q; a.kc = (const uint16_t*)k_cache; a.vc = (const uint16_t*)v_cache;
  a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.G = Hq / Hkv;
  a.scale_log2 = scale * kLog2e;
  a.num_pages = num_pages; a.P = page_size; a.W = table_width; a.table = table;
  a.lengths = own_lengths; a.max_length = max_length;
  a.items = (const Item*)items; a.rows = rows;
  a.part_at = row_parts; a.n_prefix = row_parts + Nq; a.n_part = row_parts + 2 * (int64_t)Nq;
  a.part_o = part_o; a.part_ml = (float2*)part_ml;
  hipStream_t st = (hipStream_t)stream;
  if (n_items > 0) {
    if (dtype == 0) launch_blocks<0>(a, n_items, st);
    else launch_blocks<1>(a, n_items, st);
    const int rc = moba_launch_status("shared_attention(blocks)");
    if (rc) return rc;
  }
  const bool many = max_parts > 4;
  if (dtype == 0)
    many ? launch_merge<0, 4>(a, Nq, (uint16_t*)out, lse, st) : launch_merge<0, 1>(a, Nq, (uint16_t*)out, lse, st);
  else
    many ? launch_merge<1, 4>(a, Nq, (uint16_t*)out, lse, st) : launch_merge<1, 1>(a, Nq, (uint16_t*)out, lse, st);
  return moba_launch_status("shared_attention(merge)");
}
