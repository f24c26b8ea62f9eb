// 8-bit paged KV cache on gfx950: tokens quantised as they are written, read back,
// and the chunk means that routing takes of the stored keys.  Formats, layout and
// rounding: quant.h.  The attention that reads the pool: quant_attn.hip.
//
// Append: keys turn by their positions first (as in rotary.hip: pairs (i, i + R/2) or
// (2i, 2i + 1), y_a = x_a cos - x_b sin, y_b = x_a sin + x_b cos, fp32, here with
// each product rounded), and are quantised from fp32, so that a stored key is
// rounded once.  Several lanes hold a row; the maximum of |x| goes through them.
//
// Bound by memory where tokens are many: 32K tokens of 32 + 8 + 8 heads of 128 dims, all
// turned (739 MB): 154 to 158 us, 4.7 TB/s, where a copy of 1 GiB runs at 5.1.  8 tokens of 12 +
// 2 + 2 heads: 4.2 us, a launch and what waits for each other (slot and position, page,
// store).  One pass: a row's scale is known before its values leave the registers.
#include <algorithm>

#include "quant.h"
#include "../../include/moba_hip.h"

using namespace moba;

namespace moba {
int quant_pool_of(const char* what, int format, const void* k, const void* v, const float* ks,
                  const float* vs, int num_pages, int page_size, int Hkv, int D, const int* table,
                  int B, int W, QuantPool& p) {
  if (format != 0 && format != 1) { moba_set_error("%s: format must be 0 (int8) or 1 (fp8)", what); return MOBA_ERR_ARG; }
  if (num_pages < 1 || page_size < 1 || Hkv < 1 || B < 1 || W < 1) { moba_set_error("%s: nonempty page pool and table required", what); return MOBA_ERR_ARG; }
  if (D < 8 || D > 256 || D % 8) { moba_set_error("%s: head_dim must be a multiple of 8 in [8,256]", what); return MOBA_ERR_ARG; }
  if ((int64_t)num_pages * page_size >= 1ll << 31 || (int64_t)W * page_size >= 1ll << 31) { moba_set_error("%s: page pool exceeds int32 token capacity", what); return MOBA_ERR_ARG; }
  p.Dp = code_width(D);
  // rows and 16-byte pieces of codes are counted in 32 bits: 64 GiB of codes
  if ((int64_t)num_pages * page_size * Hkv > 0xfffffff0ll / (p.Dp / 16)) { moba_set_error("%s: page pool exceeds 64 GiB of codes", what); return MOBA_ERR_ARG; }
  if ((((uintptr_t)k | (uintptr_t)v) & 15) || (((uintptr_t)ks | (uintptr_t)vs) & 3)) { moba_set_error("%s: codes must be 16-byte aligned", what); return MOBA_ERR_ARG; }
  p.k = (uint8_t*)k; p.v = (uint8_t*)v; p.ks = (float*)ks; p.vs = (float*)vs;
  p.num_pages = num_pages; p.P = page_size; p.Hkv = Hkv; p.D = D;
  p.by_page = fast_div(page_size);
  p.table = table; p.B = B; p.W = W;
  return MOBA_OK;
}
}  // namespace moba

namespace {

enum { kBadSlot = 1, kBadCell = 2, kBadAngle = 4 };

MOBA_DEV void report(int* status, int what) {
  if (status != nullptr) atomicOr(status, what);
}

// ------------------------------------------------------------------ append
struct AppendArgs {
  QuantPool pool;
  const uint16_t *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // token and head strides, elements
  int Hq, R, lanes, lanes_log, inter;          // lanes of a row, a power of two
  uint32_t rows;                               // N * (Hq + 2 Hkv)
  FastDiv by_token;                            // Hq + 2 Hkv
  const float2* cos_sin;
  int max_pos;
  const int *seq, *pos, *offsets;
  uint16_t* q_out;
  int* status;
};

// A row of work: its input, its row of angles (null: it does not turn), and where
// it goes: q_out's row (cell -1), or a cell of the pool.
struct Row {
  const uint16_t* src;
  const float2* turn;
  uint16_t* q_dst;
  int64_t cell;
  bool is_v;
};
// False: nothing of the row is written.
MOBA_DEV bool locate(const AppendArgs& a, uint32_t row, bool first_lane, Row& r) {
  const uint32_t t = div_by(row, a.by_token);
  const uint32_t h = row - t * a.by_token.d;
  const int s = a.seq[t], p = a.pos[t];
  if (s < 0 || s >= a.pool.B) {  // padding (-1), or no such slot: left as it was
    if (s != -1 && h == 0 && first_lane) report(a.status, kBadSlot);
    return false;
  }
  bool angle = true;
  r.turn = nullptr;
  if (a.cos_sin != nullptr) {
    // the table's row, in 64 bits: position + offset may pass 31
    const int64_t rp = (int64_t)p + (a.offsets != nullptr ? a.offsets[s] : 0);
    angle = rp >= 0 && rp < a.max_pos;
    if (!angle && h == 0 && first_lane) report(a.status, kBadAngle);
    r.turn = a.cos_sin + (angle ? rp : 0) * (a.R / 2);
  }
  r.cell = -1;
  r.is_v = false;
  if (h < (uint32_t)a.Hq) {
    r.src = a.q + (int64_t)t * a.q_ts + (int64_t)h * a.q_hs;
    r.q_dst = a.q_out + ((int64_t)t * a.Hq + h) * a.pool.D;
    return angle;
  }
  const uint32_t kv = h - a.Hq;
  r.is_v = kv >= (uint32_t)a.pool.Hkv;
  const int kh = (int)(r.is_v ? kv - a.pool.Hkv : kv);
  r.cell = pool_row(a.pool, s, p, kh);
  if (r.cell < 0 && kv == 0 && first_lane) report(a.status, kBadCell);
  r.src = r.is_v ? a.v + (int64_t)t * a.v_ts + (int64_t)kh * a.v_hs
                 : a.k + (int64_t)t * a.k_ts + (int64_t)kh * a.k_hs;
  if (r.is_v) r.turn = nullptr;
  return r.cell >= 0 && angle;  // a token without its angle has neither key nor value written
}

MOBA_DEV void rotate(float& x, float& y, float2 t) {
  const float a = x * t.x - y * t.y, b = x * t.y + y * t.x;
  x = a;
  y = b;
}

// The largest |x| of a row, as bits, over its lanes (on: the lane has dims of it).
template <int N> MOBA_DEV uint32_t row_max(const float (&v)[N], bool on, int lanes) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = on ? m : 0u;
  for (int off = 1; off < lanes; off <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
  return m;
}

// N codes (8 or 4) of v, from dst on.
template <int FMT, int N> MOBA_DEV void store_codes(uint8_t* dst, const float* v, const RowScale& r) {
  uint32_t w[N / 4];
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = r.finite ? to_code<FMT>(v[4 * j + i], r) : 0.0f;
    w[j] = codes4<FMT>(y[0], y[1], y[2], y[3]);
  }
  if constexpr (N == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(dst) = w[0];
}

MOBA_DEV void store_scale(const AppendArgs& a, const Row& r, float scale) {
  (r.is_v ? a.pool.vs : a.pool.ks)[r.cell] = scale;
}

// Rows of whole pieces of VEC dims (8 or 4), R a multiple of two of them (0: nothing
// turns): a lane has two pieces, those at VEC u and VEC u + R/2 of what turns, or the
// pieces c and c + n of the 2n behind R, so that a pair's two values are in one lane and
// neighbouring lanes have neighbouring pieces.  25K tokens of 12 + 2 + 2 heads of 40 dims, all
// turned: 24 us in pieces of 4, 42 where each dim finds its partner.
template <int DT, int FMT, int VEC>
__global__ __launch_bounds__(256) void append_pairs_kernel(AppendArgs a) {
  typedef uint32_t words __attribute__((ext_vector_type(VEC / 2)));
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = idx >> a.lanes_log;
  if (row >= a.rows) return;
  const int u = (int)(idx & (a.lanes - 1)), D = a.pool.D;
  Row r;
  if (!locate(a, row, u == 0, r)) return;
  const int turning = r.turn != nullptr ? a.R / (2 * VEC) : 0, from = turning * 2 * VEC;
  const int n = (D - from) / (2 * VEC), c = u - turning;
  const bool on = u < D / (2 * VEC), turns = u < turning;
  const int d0 = turns ? VEC * u : on ? from + VEC * c : 0;
  const int d1 = turns ? d0 + a.R / 2 : on ? d0 + VEC * n : 0;
  const words x = *reinterpret_cast<const words*>(r.src + d0);
  const words y = *reinterpret_cast<const words*>(r.src + d1);
  float v[2 * VEC];
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) {
    unpack2<DT>(x[i], v[2 * i], v[2 * i + 1]);
    unpack2<DT>(y[i], v[VEC + 2 * i], v[VEC + 1 + 2 * i]);
  }
  if (turns) {
    if (a.inter) {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {  // two pairs an access, as the table has them
        const float4 w = *reinterpret_cast<const float4*>(r.turn + (i < VEC / 2 ? d0 / 2 + i : d1 / 2 + i - VEC / 2));
        rotate(v[2 * i], v[2 * i + 1], make_float2(w.x, w.y));
        rotate(v[2 * i + 2], v[2 * i + 3], make_float2(w.z, w.w));
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        const float4 w = *reinterpret_cast<const float4*>(r.turn + d0 + i);
        rotate(v[i], v[VEC + i], make_float2(w.x, w.y));
        rotate(v[i + 1], v[VEC + 1 + i], make_float2(w.z, w.w));
      }
    }
  }
  if (r.cell < 0) {
    if (!on) return;
    words p, q;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      p[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
      q[i] = pack2<DT>(v[VEC + 2 * i], v[VEC + 1 + 2 * i]);
    }
    *reinterpret_cast<words*>(r.q_dst + d0) = p;
    *reinterpret_cast<words*>(r.q_dst + d1) = q;
    return;
  }
  const RowScale s = row_scale<FMT>(row_max(v, on, a.lanes));
  uint8_t* dst = (r.is_v ? a.pool.v : a.pool.k) + r.cell * a.pool.Dp;
  if (u == 0) {
    store_scale(a, r, s.scale);
    if (D < a.pool.Dp) *reinterpret_cast<uint2*>(dst + D) = make_uint2(0, 0);  // behind D
  }
  if (!on) return;
  store_codes<FMT, VEC>(dst + d0, v, s);
  store_codes<FMT, VEC>(dst + d1, v + VEC, s);
}

// Any other row: a lane has 8 neighbouring dims and reads the partner of each one
// that turns by itself.  WIDE: rows are whole 16-byte pieces.
template <int DT, int FMT, bool WIDE>
__global__ __launch_bounds__(256) void append_any_kernel(AppendArgs a) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  const uint32_t row = idx >> a.lanes_log;
  if (row >= a.rows) return;
  const int u = (int)(idx & (a.lanes - 1)), D = a.pool.D, half = a.R / 2;
  Row r;
  if (!locate(a, row, u == 0, r)) return;
  const bool on = 8 * u < D;
  const int d = on ? 8 * u : 0;
  float v[8];
  if constexpr (WIDE) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(r.src + d);
#pragma unroll
    for (int i = 0; i < 4; ++i) unpack2<DT>(x[i], v[2 * i], v[2 * i + 1]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32<DT>(r.src[d + e]);
  }
  if (r.turn != nullptr && d < a.R) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int de = d + e;
      if (de >= a.R) continue;
      const bool second = a.inter ? de & 1 : de >= half;
      const int other = a.inter ? de ^ 1 : (second ? de - half : de + half);
      const float2 t = r.turn[a.inter ? de >> 1 : (second ? de - half : de)];
      float mine = v[e], theirs = to_f32<DT>(r.src[other]);
      if (second) rotate(theirs, mine, t);
      else rotate(mine, theirs, t);
      v[e] = mine;
    }
  }
  if (r.cell < 0) {
    if (!on) return;
    if constexpr (WIDE) {
      st8(r.q_dst + d, pack8<DT>(v));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) r.q_dst[d + e] = from_f32<DT>(v[e]);
    }
    return;
  }
  const RowScale s = row_scale<FMT>(row_max(v, on, a.lanes));
  if (u == 0) store_scale(a, r, s.scale);
  uint8_t* dst = (r.is_v ? a.pool.v : a.pool.k) + r.cell * a.pool.Dp;
  if (on) store_codes<FMT, 8>(dst + d, v, s);
  else if (8 * u < a.pool.Dp) *reinterpret_cast<uint2*>(dst + 8 * u) = make_uint2(0, 0);  // behind D
}

// Pieces as wide as rows and R allow; else each dim finds its partner.
template <int DT, int FMT> void launch_append(AppendArgs& a, bool wide, hipStream_t st) {
  const int D = a.pool.D;
  const int vec = !wide ? 0 : D % 16 == 0 && a.R % 16 == 0 ? 8 : a.R % 8 == 0 ? 4 : 0;
  const int units = vec ? D / (2 * vec) : a.pool.Dp / 8;
  a.lanes_log = 0;
  while ((1 << a.lanes_log) < units) ++a.lanes_log;
  a.lanes = 1 << a.lanes_log;
  const dim3 grid((unsigned)(((uint64_t)a.rows * a.lanes + 255) / 256)), block(256);
  if (vec == 8) hipLaunchKernelGGL((append_pairs_kernel<DT, FMT, 8>), grid, block, 0, st, a);
  else if (vec == 4) hipLaunchKernelGGL((append_pairs_kernel<DT, FMT, 4>), grid, block, 0, st, a);
  else if (wide) hipLaunchKernelGGL((append_any_kernel<DT, FMT, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((append_any_kernel<DT, FMT, false>), grid, block, 0, st, a);
}

// Whether every row begins at a 16-byte border.
bool whole_pieces(const void* p, int64_t ts, int64_t hs) {
  return (uintptr_t)p % 16 == 0 && ts % 8 == 0 && hs % 8 == 0;
}

// -------------------------------------------------------------------- read
struct ReadArgs {
  QuantPool pool;
  uint32_t total;  // N * Hkv * (D / 8) pieces of 8 codes
  FastDiv by_row, by_token;
  const int *seq, *pos;
  uint16_t *k_out, *v_out;
  int* status;
};

template <int DT, int FMT> MOBA_DEV void store_values(uint16_t* dst, uint2 w, float scale) {
  float x[4], y[4], v[8];
  numbers4<FMT>(w.x, x);
  numbers4<FMT>(w.y, y);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = x[i] * scale;
    v[4 + i] = y[i] * scale;
  }
  st8(dst, pack8<DT>(v));
}

// A thread has 8 dims of a token's key and of its value: one search for both.  32K tokens
// of 8 heads of 128 dims (204 MB): 39 us, 5.2 TB/s (a call 45; with key and value in threads
// of their own 66).  Stores that pass the caches by took 33, but the reader
// of the output, which comes next, would then find nothing of it there.
template <int DT, int FMT>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= a.total) return;
  const uint32_t row = div_by(idx, a.by_row), u = idx - row * a.by_row.d;
  const uint32_t t = div_by(row, a.by_token);
  const int kh = (int)(row - t * a.by_token.d), s = a.seq[t];
  const int64_t cell = pool_row(a.pool, s, a.pos[t], kh);
  const int64_t to = (int64_t)row * a.pool.D + 8 * u;
  if (cell < 0) {  // padding, or no such cell: zeros
    if (s != -1 && kh == 0 && u == 0) report(a.status, s < 0 || s >= a.pool.B ? kBadSlot : kBadCell);
    st8(a.k_out + to, zero8());
    st8(a.v_out + to, zero8());
    return;
  }
  const int64_t from = cell * a.pool.Dp + 8 * u;
  const uint2 k = *reinterpret_cast<const uint2*>(a.pool.k + from);
  const uint2 v = *reinterpret_cast<const uint2*>(a.pool.v + from);
  const float ks = a.pool.ks[cell], vs = a.pool.vs[cell];
  store_values<DT, FMT>(a.k_out + to, k, ks);
  store_values<DT, FMT>(a.v_out + to, v, vs);
}

// ------------------------------------------------------------------- means
constexpr int kMeansPer = 16;  // tokens of a lane: chunks of up to 1024

// One wave per (item, kv head, 8 dims): lane j sums the stored numbers of tokens
// j, j + 64, ... in order, then canon_tree, as the 16-bit cache's means do.  All
// lookups, then all loads, then the sums; a token without a cell adds nothing.
// A wave of modest size: a chunk closes once in `chunk` tokens.
template <int DT, int FMT>
__global__ __launch_bounds__(64) void means_kernel(QuantPool p, const int* __restrict__ seq,
                                                   const int* __restrict__ chunk_or_pos, int mode,
                                                   int C, uint16_t* __restrict__ means,
                                                   int max_chunks) {
  const int nd = p.D / 8, db = blockIdx.x % nd, kh = (blockIdx.x / nd) % p.Hkv;
  const int i = blockIdx.x / (nd * p.Hkv), lane = threadIdx.x;
  const int sid = seq[i];
  int chunk = chunk_or_pos[i];
  if (mode == 1) {
    if ((chunk + 1) % C != 0) return;
    chunk = chunk / C;
  }
  if (sid < 0 || sid >= p.B || chunk < 0 || chunk >= max_chunks) return;
  int64_t row[kMeansPer];
#pragma unroll
  for (int k = 0; k < kMeansPer; ++k) {
    const int j = lane + 64 * k;
    row[k] = j < C ? pool_row(p, sid, chunk * C + j, kh) : -1;
  }
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.0f;
#pragma unroll
  for (int k = 0; k < kMeansPer; ++k) {
    const int64_t at = row[k] >= 0 ? row[k] : 0;
    const uint2 w = *reinterpret_cast<const uint2*>(p.k + at * p.Dp + 8 * db);
    const float scale = p.ks[at];
    float x[4], y[4];
    numbers4<FMT>(w.x, x);
    numbers4<FMT>(w.y, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[e] += row[k] >= 0 ? x[e] * scale : 0.0f;
      acc[4 + e] += row[k] >= 0 ? y[e] * scale : 0.0f;
    }
  }
  uint16_t res[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) res[e] = from_f32<DT>(canon_tree(acc[e]) / (float)C);
  if (lane == 0) {
    uint16_t* dst = means + (((int64_t)sid * max_chunks + chunk) * p.Hkv + kh) * p.D + 8 * db;
#pragma unroll
    for (int e = 0; e < 8; ++e) dst[e] = res[e];
  }
}

}  // namespace

extern "C" int moba_hip_quantized_append(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                         const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                         const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                         int dtype, int N, int Hq, int Hkv, int D,
                                         const float* cos_sin, int max_pos, int rotary_dim,
                                         int interleaved, int format, void* k_codes, void* v_codes,
                                         float* k_scale, float* v_scale, int num_pages, int page_size,
                                         const int* table, int B, int table_width,
                                         const int* token_seq, const int* token_pos,
                                         const int* offsets, void* q_out, int* status, void* stream) {
  AppendArgs a;
  const int rc = quant_pool_of("quantized_append", format, k_codes, v_codes, k_scale, v_scale, num_pages,
                               page_size, Hkv, D, table, B, table_width, a.pool);
  if (rc) return rc;
  if (dtype != 0 && dtype != 1) { moba_set_error("quantized_append: dtype must be 0 (bf16) or 1 (fp16)"); return MOBA_ERR_ARG; }
  if (N < 1 || Hq < 0) { moba_set_error("quantized_append: nonempty N required"); return MOBA_ERR_ARG; }
  if (cos_sin != nullptr && (rotary_dim < 2 || rotary_dim > D || rotary_dim % 2 || max_pos < 1)) { moba_set_error("quantized_append: rotary_dim must be even, in [2, D], and the table nonempty"); return MOBA_ERR_ARG; }
  if ((uintptr_t)cos_sin & 15) { moba_set_error("quantized_append: the cos / sin table must be 16-byte aligned"); return MOBA_ERR_ARG; }
  if ((Hq > 0) != (q != nullptr) || (Hq > 0) != (q_out != nullptr) || (Hq > 0 && cos_sin == nullptr)) { moba_set_error("quantized_append: q, q_out and the cos / sin table go together with Hq > 0"); return MOBA_ERR_ARG; }
  // 8 elements a lane, lanes of a row rounded up to a power of two: a launch of 2^31 threads
  if ((int64_t)N * (Hq + 2ll * Hkv) * a.pool.Dp >= 1ll << 33) { moba_set_error("quantized_append: more than 2^33 elements in one call"); return MOBA_ERR_ARG; }
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.q_ts = q_token_stride; a.q_hs = q_head_stride;
  a.k_ts = k_token_stride; a.k_hs = k_head_stride;
  a.v_ts = v_token_stride; a.v_hs = v_head_stride;
  a.Hq = Hq; a.R = cos_sin != nullptr ? rotary_dim : 0; a.inter = interleaved;
  a.by_token = fast_div(Hq + 2 * Hkv);
  a.rows = (uint32_t)N * a.by_token.d;
  a.cos_sin = (const float2*)cos_sin; a.max_pos = max_pos;
  a.seq = token_seq; a.pos = token_pos; a.offsets = offsets;
  a.q_out = (uint16_t*)q_out; a.status = status;
  const bool wide = whole_pieces(k, a.k_ts, a.k_hs) && whole_pieces(v, a.v_ts, a.v_hs) &&
                    (Hq == 0 || (whole_pieces(q, a.q_ts, a.q_hs) && whole_pieces(q_out, 0, 0)));
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0) { if (format == 0) launch_append<0, 0>(a, wide, st); else launch_append<0, 1>(a, wide, st); }
  else { if (format == 0) launch_append<1, 0>(a, wide, st); else launch_append<1, 1>(a, wide, st); }
  return moba_launch_status("quantized_append");
}

extern "C" int moba_hip_quantized_read(int format, const void* k_codes, const void* v_codes,
                                       const float* k_scale, const float* v_scale, int num_pages,
                                       int page_size, int Hkv, int D, const int* table, int B,
                                       int table_width, const int* token_seq, const int* token_pos,
                                       int N, int dtype, void* k_out, void* v_out, int* status,
                                       void* stream) {
  ReadArgs a;
  const int rc = quant_pool_of("quantized_read", format, k_codes, v_codes, k_scale, v_scale, num_pages,
                               page_size, Hkv, D, table, B, table_width, a.pool);
  if (rc) return rc;
  if (dtype != 0 && dtype != 1) { moba_set_error("quantized_read: dtype must be 0 (bf16) or 1 (fp16)"); return MOBA_ERR_ARG; }
  if (N < 1) { moba_set_error("quantized_read: nonempty N required"); return MOBA_ERR_ARG; }
  if (((uintptr_t)k_out | (uintptr_t)v_out) & 15) { moba_set_error("quantized_read: outputs must be 16-byte aligned"); return MOBA_ERR_ARG; }
  if ((int64_t)N * Hkv * (D / 8) >= 1ll << 31) { moba_set_error("quantized_read: more than 2^31 pieces of 8 elements in one call"); return MOBA_ERR_ARG; }
  a.by_row = fast_div(D / 8);
  a.by_token = fast_div(Hkv);
  a.total = (uint32_t)N * Hkv * (D / 8);
  a.seq = token_seq; a.pos = token_pos;
  a.k_out = (uint16_t*)k_out; a.v_out = (uint16_t*)v_out; a.status = status;
  const dim3 grid((a.total + 255) / 256), block(256);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == 0 && format == 0) hipLaunchKernelGGL((read_kernel<0, 0>), grid, block, 0, st, a);
  else if (dtype == 0) hipLaunchKernelGGL((read_kernel<0, 1>), grid, block, 0, st, a);
  else if (format == 0) hipLaunchKernelGGL((read_kernel<1, 0>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((read_kernel<1, 1>), grid, block, 0, st, a);
  return moba_launch_status("quantized_read");
}

extern "C" int moba_hip_quantized_means(int format, const void* k_codes, const float* k_scale,
                                        int num_pages, int page_size, int Hkv, int D, const int* table,
                                        int B, int table_width, const int* item_seq,
                                        const int* item_chunk_or_pos, int n_items, int mode, int chunk,
                                        int dtype, void* means, int max_chunks, void* stream) {
  if (n_items <= 0) return MOBA_OK;
  QuantPool p;
  const int rc = quant_pool_of("quantized_means", format, k_codes, k_codes, k_scale, k_scale, num_pages,
                               page_size, Hkv, D, table, B, table_width, p);
  if (rc) return rc;
  if (dtype != 0 && dtype != 1) { moba_set_error("quantized_means: dtype must be 0 (bf16) or 1 (fp16)"); return MOBA_ERR_ARG; }
  if (chunk < 1 || chunk > 64 * kMeansPer || max_chunks < 1) { moba_set_error("quantized_means: chunk must be in [1,1024], the means nonempty"); return MOBA_ERR_ARG; }
  const int64_t per_item = (int64_t)Hkv * (D / 8);
  const int most = (int)(((1ll << 26) - 1) / per_item);  // items of a launch: 2^32 threads are too many
  if (n_items * per_item >= 1ll << 31 || most < 1 || (int64_t)max_chunks * chunk >= 1ll << 31) { moba_set_error("quantized_means: more than 2^31 pieces or positions, or 2^26 pieces of an item"); return MOBA_ERR_ARG; }
  hipStream_t st = (hipStream_t)stream;
#define MOBA_MEANS(DT_, FMT_)                                                                      \
  hipLaunchKernelGGL((means_kernel<DT_, FMT_>), grid, block, 0, st, p, item_seq + at,               \
                     item_chunk_or_pos + at, mode, chunk, (uint16_t*)means, max_chunks)
  for (int at = 0; at < n_items; at += std::min(most, n_items - at)) {
    const dim3 grid((unsigned)(std::min(most, n_items - at) * per_item)), block(64);
    if (dtype == 0) { if (format == 0) MOBA_MEANS(0, 0); else MOBA_MEANS(0, 1); }
    else { if (format == 0) MOBA_MEANS(1, 0); else MOBA_MEANS(1, 1); }
  }
#undef MOBA_MEANS
  return moba_launch_status("quantized_means");
}
