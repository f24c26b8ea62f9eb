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
__device__ __attribute__((aligned(512))) const uint16_t g_zero[256] = {0};

// 16 bytes per lane from any address straight into LDS (lane l's at
// lds + 16 l); ordered by the caller as dma_lds16.
MOBA_DEV void dma_global16(const void* p, const void* lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :: "s"(lds_addr(lds)), "v"(p) : "memory", "m0");
}

template <int DT, int ND>
__global__ __launch_bounds__(256, 2) void block_kernel(SharedArgs a) {
  constexpr int DP = ND <= 64 ? 64 : ND <= 128 ? 128 : 256;  // row of the LDS layout
  constexpr int NKS = ND / 16, NDB = ND / 32;
  constexpr int KEYS = DP <= 64 ? 64 : 32, NKB = KEYS / 32;
  constexpr int TILE = KEYS * DP, NB = DP / 8, NDMA = KEYS * NB / 256;
  constexpr int TPC = 256 / KEYS;   // tiles per 256 looked-up tokens
  __shared__ __attribute__((aligned(16))) uint16_t Ks[2][TILE];
  __shared__ __attribute__((aligned(16))) uint16_t Vs[2][TILE];
  __shared__ __attribute__((aligned(16))) uint32_t tok[2][256];  // pool token of each key
  __shared__ int holes[2][4];                                    // of 64 keys, any has none
  __shared__ int wmax[4];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qi = lane & 31, hh = lane >> 5;
  const Item x = a.items[blockIdx.x];
  if (x.n_m == 0) return;
  const int D = a.D;

  const int m = wave * 32 + qi;
  const bool valid = m < x.n_m;
  const int pair = x.m0 + min(m, x.n_m - 1);
  const int row = a.rows[x.row_at + pair / a.G];
  const int h = x.kh * a.G + pair % a.G;
  int limit = x.length, length = x.length;
  if (x.length < 0) {
    limit = max(0, min(a.lengths[row], a.max_length));
    int mx = limit;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = max(mx, __shfl_xor(mx, o, 64));
    if (lane == 0) wmax[wave] = mx;
    __syncthreads();
    length = max(max(wmax[0], wmax[1]), max(wmax[2], wmax[3]));
  }
  // the split's keys: whole groups of 64 but for the last
  const int per = ((length + 64 * x.splits - 1) / (64 * x.splits)) * 64;
  const int lo = min(length, x.split * per), hi = min(length, lo + per);
  const int64_t slot = ((int64_t)a.part_at[row] + (x.length < 0 ? a.n_prefix[row] : 0) + x.split) *
                       a.Hq + h;
  if (lo >= hi) {
    if (valid && hh == 0) a.part_ml[slot] = make_float2(-INFINITY, 0.0f);
    return;
  }

  const int* trow = a.table + (int64_t)x.slot * a.W;
  auto lookup = [&](int c) -> uint32_t {  // this thread's key of 256
    const int key = lo + c * 256 + tid;
    if (key >= hi) return kNoToken;
    const int lp = key / a.P, page = trow[lp];
    return page >= 0 && page < a.num_pages ? (uint32_t)page * a.P + (key - lp * a.P) : kNoToken;
  };
  auto publish = [&](int c, uint32_t t) {
    tok[c & 1][tid] = t;
    const bool any = __any(t == kNoToken);
    if (lane == 0) holes[c & 1][wave] = any;
  };
  const char *kp = (const char*)(a.kc + (int64_t)x.kh * D), *vp = (const char*)(a.vc + (int64_t)x.kh * D);
  const int64_t row_bytes = (int64_t)a.Hkv * D * 2;
  // thread (wave w, lane l) brings 16-byte blocks j = (n * 4 + w) * 64 + l of a
  // tile: row j / NB, physical block j % NB of the swizzled row
  auto dma = [&](int it) {
    const uint32_t* tk = &tok[(it / TPC) & 1][(it % TPC) * KEYS];
#pragma unroll
    for (int n = 0; n < NDMA; ++n) {
      const int j = (n * 4 + wave) * 64 + lane, r = j / NB;
      const int col = swz<DP>(r, (j % NB) * 8) - r * DP;
      if (col < ND) {
        const uint32_t t = tk[r];
        const bool on = t != kNoToken && col < D;
        const int64_t off = (int64_t)t * row_bytes + col * 2;
        const char* z = (const char*)(g_zero + col);
        dma_global16(on ? kp + off : z, &Ks[it & 1][(n * 4 + wave) * 64 * 8]);
        dma_global16(on ? vp + off : z, &Vs[it & 1][(n * 4 + wave) * 64 * 8]);
      }
    }
  };

  publish(0, lookup(0));
  u16x8_t qf[NKS];
  const uint16_t* qrow = a.q + ((int64_t)row * a.Hq + h) * D;
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
  const float c2 = a.scale_log2;
  const bool idle = wave * 32 >= x.n_m;
  int wlim = valid ? limit : 0x7fffffff;  // the wave's shortest row
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) wlim = min(wlim, __shfl_xor(wlim, o, 64));
  wlim = __builtin_amdgcn_readfirstlane(wlim);

  const uint32_t kbase0 = swz_b128_base<DP>(lane);
  const uint32_t trb0 = swz_tr_base<DP>(lane, 0), trb1 = swz_tr_base<DP>(lane, 1);
  auto tile = [&](int it) {
    const uint16_t *Kb = Ks[it & 1], *Vb = Vs[it & 1];
    const int kt0 = lo + it * KEYS;
    f32x16_t sacc[NKB];
    wave_prio<1>();
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
      sacc[kb] = zero16();
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
        sacc[kb] = mfma32<DT>(lds8(Kb, kb * 32 * DP * 2 + swz_b128<DP>(kbase0, ks)), qf[ks], sacc[kb]);
    }
    wave_prio<0>();
    const int at = (it % TPC) * KEYS, c = (it / TPC) & 1;
    if (kt0 + KEYS > wlim || holes[c][at / 64]) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int k = kb * 32 + 8 * (r >> 2) + 4 * hh + (r & 3);
          const bool ok = kt0 + k < limit && tok[c][at + k] != kNoToken;
          sacc[kb][r] = ok ? sacc[kb][r] : -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sacc[kb][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c2;
    const bool up = mx > m_run;
    if (__any(up)) {
      const float mn = up ? mx : m_run;
      const float alpha = up ? fast_exp2(m_run - mn) : 1.0f;
      lsum *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[db][r] *= alpha;
      m_run = mn;
    }
    // a row with nothing so far: weights of 0, not of exp2(-inf + inf)
    const float nm = m_run == -INFINITY ? 0.0f : -m_run;
    float ps = 0.0f;
    u16x8_t pv[NKB][2];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) {
      float p[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = fast_exp2(fmaf(sacc[kb][r], c2, nm));
        ps += p[r];
      }
      pv[kb][0] = pack8<DT>(p);
      pv[kb][1] = pack8<DT>(p + 8);
    }
    lsum += ps;
    wave_prio<1>();
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint32_t ro = (kb * 32 + t * 16) * DP * 2;
          oacc[db] = mfma32<DT>(lds_tr8(Vb, ro + swz_tr<DP>(trb0, db), ro + swz_tr<DP>(trb1, db)),
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
    if (more) next = lookup(it / TPC + 1);
    if (it + 1 < ntiles) dma(it + 1);
    if (!idle) tile(it);
    if (more) publish(it / TPC + 1, next);  // read from tile it + TPC - 1 on
  }

  const float l = lsum + __shfl_xor(lsum, 32, 64);
  if (!valid) return;
  float* po = a.part_o + slot * D;
#pragma unroll
  for (int db = 0; db < NDB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = db * 32 + 8 * j + 4 * hh;
      if (d < D)
        *reinterpret_cast<f32x4_t*>(po + d) = (f32x4_t){oacc[db][4 * j], oacc[db][4 * j + 1],
                                                        oacc[db][4 * j + 2], oacc[db][4 * j + 3]};
    }
  if (hh == 0) a.part_ml[slot] = make_float2(m_run, l);
}

// Joins the ranges of each (row, head): four dims per thread.
template <int DT>
__global__ __launch_bounds__(256) void merge_kernel(const float* __restrict__ part_o,
                                                    const float2* __restrict__ part_ml,
                                                    const int* __restrict__ part_at,
                                                    const int* __restrict__ n_part, int n_rows,
                                                    int Hq, int D, uint16_t* __restrict__ out,
                                                    float* __restrict__ lse) {
  const int tpr = D / 4, per = 256 / tpr;  // (row, head) pairs per workgroup
  const int e = threadIdx.x / tpr, d = (threadIdx.x - e * tpr) * 4;
  const int64_t rh = (int64_t)blockIdx.x * per + e;
  if (e >= per || rh >= (int64_t)n_rows * Hq) return;
  const int row = (int)(rh / Hq), h = (int)(rh - (int64_t)row * Hq);
  const int n = n_part[row];
  const int64_t s0 = (int64_t)part_at[row] * Hq + h;
  float M = -INFINITY;
  for (int i = 0; i < n; ++i) {
    const float2 ml = part_ml[s0 + (int64_t)i * Hq];
    if (ml.y != 0.0f) M = fmaxf(M, ml.x);
  }
  float z = 0.0f;
  f32x4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < n; ++i) {
    const int64_t s = s0 + (int64_t)i * Hq;
    const float2 ml = part_ml[s];
    if (ml.y == 0.0f) continue;  // an empty range wrote no O
    const float w = fast_exp2(ml.x - M);
    const f32x4_t p = *reinterpret_cast<const f32x4_t*>(part_o + s * D + d);
    z += w * ml.y;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] += w * p[k];
  }
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

}  // namespace

extern "C" int moba_hip_shared_attention(const void* q, int dtype, int Nq, int Hq, int Hkv, int D,
                                         float scale, const void* k_cache, const void* v_cache,
                                         int num_pages, int page_size, const int* table,
                                         int table_width, const int* own_lengths, int max_length,
                                         const int* items, int n_items, const int* rows,
                                         const int* row_parts, float* part_o, float* part_ml,
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
  const int per = 256 / (D / 4);
  const dim3 grid((unsigned)(((int64_t)Nq * Hq + per - 1) / per));
  if (dtype == 0)
    hipLaunchKernelGGL((merge_kernel<0>), grid, dim3(256), 0, st, part_o, a.part_ml, a.part_at, a.n_part, Nq, Hq, D, (uint16_t*)out, lse);
  else
    hipLaunchKernelGGL((merge_kernel<1>), grid, dim3(256), 0, st, part_o, a.part_ml, a.part_at, a.n_part, Nq, Hq, D, (uint16_t*)out, lse);
  return moba_launch_status("shared_attention(merge)");
}
