// Rotary append on gfx950: new keys and values go into the page pool, the keys
// rotated by their positions on the way and the queries of the same tokens
// with them, in one launch.
//
// A pair (x_a, x_b) of a head's first R dims turns by the angle p * theta_i of
// its position p:
//   y_a = x_a cos - x_b sin,   y_b = x_a sin + x_b cos
// with (a, b) = (i, i + R/2), or (2i, 2i + 1) when interleaved.  Dims from R on
// and the values are copied bit for bit.  cos and sin come from a table
// [max_pos][R/2] of fp32 pairs; the rotation is fp32 (the first product of
// each component fused into the sum), rounded once to the 16-bit type.
//
// Bound by memory: every input is read once and every output written once; the
// table's row is shared by all the heads of a token and stays in L1 / L2.  A
// 32K-token prompt of 32 + 8 + 8 heads of 128 dims (822 MB with the table): 143
// us, 5.7 TB/s (a copy of 2 GiB: 4.9); 8 tokens: 3 us, what a launch takes.
#include <algorithm>

#include "common.h"
#include "../../include/moba_hip.h"

using namespace moba;

namespace {

struct AppendArgs {
  const uint16_t *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // token and head strides, elements
  int N, Hq, Hkv, D, R, units;                 // units: pieces of work per head
  int wide;                                    // what is copied is whole 16-byte pieces
  uint32_t total;                              // N * (Hq + 2 Hkv) * units
  FastDiv by_token, by_head, by_page;
  const float2* cos_sin;
  int max_pos;
  uint16_t *kc, *vc;
  int num_pages, P;
  const int* table;
  int B, W;
  const int *seq, *pos, *offsets;
  uint16_t* q_out;
  int* status;
};

enum { kBadSlot = 1, kBadCell = 2, kBadAngle = 4 };

MOBA_DEV void report(const AppendArgs& a, int what) {
  if (a.status != nullptr) atomicOr(a.status, what);
}

// One unit of work: (token, head, piece).  The heads of a token are numbered
// q, k, v.  Returns false when the unit has nothing to write; else src and
// dst are the head's rows and turn the table row of a rotated head (null for a
// value).
MOBA_DEV bool locate(const AppendArgs& a, uint32_t idx, int& unit, const uint16_t*& src,
                     uint16_t*& dst, const float2*& turn) {
  const uint32_t t = div_by(idx, a.by_token);
  const uint32_t in = idx - t * a.by_token.d;
  const uint32_t h = div_by(in, a.by_head);
  unit = (int)(in - h * a.by_head.d);
  const int s = a.seq[t], p = a.pos[t];
  if (s < 0 || s >= a.B) {  // padding (-1), or no such slot: left as it was
    if (s != -1 && in == 0) report(a, kBadSlot);
    return false;
  }
  // the table's row, in 64 bits: position + offset may pass 31
  const int64_t rp = (int64_t)p + (a.offsets != nullptr ? a.offsets[s] : 0);
  const bool angle = rp >= 0 && rp < a.max_pos;
  if (!angle && in == 0) report(a, kBadAngle);
  turn = a.cos_sin + (angle ? rp : 0) * (a.R / 2);
  if (h < (uint32_t)a.Hq) {
    src = a.q + (int64_t)t * a.q_ts + (int64_t)h * a.q_hs;
    dst = a.q_out + ((int64_t)t * a.Hq + h) * a.D;
    return angle;
  }
  const uint32_t lp = p >= 0 ? div_by((uint32_t)p, a.by_page) : (uint32_t)a.W;
  const int page = lp < (uint32_t)a.W ? a.table[(int64_t)s * a.W + lp] : -1;
  const bool cell = page >= 0 && page < a.num_pages;
  uint32_t kh = h - a.Hq;
  if (!cell && kh == 0 && unit == 0) report(a, kBadCell);
  const bool is_v = kh >= (uint32_t)a.Hkv;
  if (is_v) kh -= a.Hkv;
  const int64_t row = (int64_t)page * a.P + (p - (int)(lp * a.by_page.d));
  dst = (is_v ? a.vc : a.kc) + (row * a.Hkv + kh) * a.D;
  src = is_v ? a.v + (int64_t)t * a.v_ts + (int64_t)kh * a.v_hs
             : a.k + (int64_t)t * a.k_ts + (int64_t)kh * a.k_hs;
  if (is_v) turn = nullptr;
  return cell && angle;  // a token without its angle has neither key nor value written
}

MOBA_DEV void rotate(float x, float y, float2 t, float& xo, float& yo) {
  const float a = fmaf(x, t.x, -(y * t.y)), b = fmaf(x, t.y, y * t.x);
  xo = a;
  yo = b;
}

// VEC 16-bit values of a row as one access (16, 8 or 4 bytes).
template <int VEC> struct Piece {
  typedef uint32_t words __attribute__((ext_vector_type(VEC / 2)));
  words w;
  MOBA_DEV void load(const uint16_t* p) { w = *reinterpret_cast<const words*>(p); }
  MOBA_DEV void store(uint16_t* p) const { *reinterpret_cast<words*>(p) = w; }
};
template <> struct Piece<2> {
  uint32_t w[1];
  MOBA_DEV void load(const uint16_t* p) { w[0] = *reinterpret_cast<const uint32_t*>(p); }
  MOBA_DEV void store(uint16_t* p) const { *reinterpret_cast<uint32_t*>(p) = w[0]; }
};

// The pieces c and c + n of the 2n of VEC dims from `from` on.
template <int VEC> MOBA_DEV void copy_pieces(const AppendArgs& a, const uint16_t* src, uint16_t* dst, int from, int c) {
  const int n = (a.D - from + 2 * VEC - 1) / (2 * VEC), d0 = from + VEC * c, d1 = d0 + VEC * n;
  if (c >= n) return;
  Piece<VEC> x, y;
  x.load(src + d0);
  y.load(src + (d1 < a.D ? d1 : d0));
  x.store(dst + d0);
  if (d1 < a.D) y.store(dst + d1);
}

// Whole pieces of VEC dims, two per unit, so that neighbouring lanes have
// neighbouring pieces in each of the two accesses: unit u < R / 2 VEC turns the
// pieces at VEC u and VEC u + R/2 (VEC pairs of the two, or VEC / 2 pairs within
// each when interleaved), unit R / 2 VEC + c copies the pieces c and c + n of
// the 2n behind R.  8K tokens, 16 + 4 + 4 heads: of 40 dims, all rotated, 10.3 us
// in 8-byte pieces, 17.3 dim by dim; of 256 dims, 24 rotated, 44 with the others in
// 16-byte pieces (wide), 54 in 8-byte ones too; 64 rotated, 40, 45 where a unit has
// two neighbouring pieces.
template <int DT, bool INTER, int VEC>
__global__ __launch_bounds__(256) void append_pairs_kernel(AppendArgs a) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= a.total) return;
  int u;
  const uint16_t* src;
  uint16_t* dst;
  const float2* turn;
  if (!locate(a, idx, u, src, dst, turn)) return;
  const int turning = turn != nullptr ? a.R / (2 * VEC) : 0, from = turning * 2 * VEC;
  Piece<VEC> x, y;
  if (u >= turning) {
    if (VEC < 8 && a.wide) copy_pieces<8>(a, src, dst, from, u - turning);
    else copy_pieces<VEC>(a, src, dst, from, u - turning);
    return;
  }
  const int d0 = VEC * u, d1 = d0 + a.R / 2;
  x.load(src + d0);
  y.load(src + d1);
  float2 t[VEC];
#pragma unroll
  for (int i = 0; i < VEC; i += 2) {  // two pairs an access, as the table has them
    const int pair = !INTER ? d0 + i : i < VEC / 2 ? d0 / 2 + i : d1 / 2 + i - VEC / 2;
    if constexpr (INTER && VEC == 2) {
      t[0] = turn[d0 / 2];
      t[1] = turn[d1 / 2];
    } else {
      const float4 w = *reinterpret_cast<const float4*>(turn + pair);
      t[i] = make_float2(w.x, w.y);
      t[i + 1] = make_float2(w.z, w.w);
    }
  }
  float v[2 * VEC];
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) {
    unpack2<DT>(x.w[i], v[2 * i], v[2 * i + 1]);
    unpack2<DT>(y.w[i], v[VEC + 2 * i], v[VEC + 2 * i + 1]);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float& p = INTER ? v[2 * i] : v[i];
    float& q = INTER ? v[2 * i + 1] : v[VEC + i];
    rotate(p, q, t[i], p, q);
  }
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) {
    x.w[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
    y.w[i] = pack2<DT>(v[VEC + 2 * i], v[VEC + 2 * i + 1]);
  }
  x.store(dst + d0);
  y.store(dst + d1);
}

// Any even R: unit u writes dims VEC u .. VEC u + VEC - 1, and reads the
// partner of each rotated one by itself.  VEC 8 where rows are whole 16-byte
// pieces, else 1.
template <int DT, int VEC>
__global__ __launch_bounds__(256) void append_any_kernel(AppendArgs a, int inter) {
  const uint32_t idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= a.total) return;
  int u;
  const uint16_t* src;
  uint16_t* dst;
  const float2* turn;
  if (!locate(a, idx, u, src, dst, turn)) return;
  const int d = VEC * u, half = a.R / 2;
  uint16_t x[VEC];
  if constexpr (VEC == 8) {
    const u16x8_t w = ld8(src + d);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = w[e];
  } else {
    x[0] = src[d];
  }
  if (turn != nullptr && d < a.R) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int de = d + e;
      if (de >= a.R) continue;
      const bool second = inter ? de & 1 : de >= half;
      const int other = inter ? de ^ 1 : (second ? de - half : de + half);
      const float2 t = turn[inter ? de >> 1 : (second ? de - half : de)];
      const float mine = to_f32<DT>(x[e]), theirs = to_f32<DT>(src[other]);
      float lo, hi;
      rotate(second ? theirs : mine, second ? mine : theirs, t, lo, hi);
      x[e] = from_f32<DT>(second ? hi : lo);
    }
  }
  if constexpr (VEC == 8) {
    u16x8_t w;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = x[e];
    st8(dst + d, w);
  } else {
    dst[d] = x[0];
  }
}

// Widest access that every row allows: 8, 4, 2 or 1 dims.
int row_access(const void* p, int64_t ts, int64_t hs, int D) {
  const uint64_t bits = ((uint64_t)(uintptr_t)p >> 1) | (uint64_t)ts | (uint64_t)hs | (uint64_t)D;
  return ((uintptr_t)p & 1) ? 1 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
}

template <int DT, int VEC> void launch_pairs(AppendArgs& a, int interleaved, hipStream_t st) {
  const dim3 grid((a.total + 255) / 256), block(256);
  if (interleaved) hipLaunchKernelGGL((append_pairs_kernel<DT, true, VEC>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((append_pairs_kernel<DT, false, VEC>), grid, block, 0, st, a);
}

// access: of the rows.  Pairs in whole pieces where R / 2 dims are whole pieces
// too; else each dim finds its partner.
template <int DT>
void launch_append(AppendArgs& a, int interleaved, int access, hipStream_t st) {
  int vec = access;
  while (vec > 1 && a.R % (2 * vec)) vec /= 2;
  const bool pairs = vec > 1;
  a.wide = access == 8 && a.R % 8 == 0;
  const int copy = a.wide ? 16 : 2 * vec;  // dims that a unit copies
  a.units = pairs ? a.R / (2 * vec) + (a.D - a.R + copy - 1) / copy : access == 8 ? a.D / 8 : a.D;
  a.by_head = fast_div(a.units);
  a.by_token = fast_div((a.Hq + 2 * a.Hkv) * a.units);
  a.total = (uint32_t)a.N * a.by_token.d;
  const dim3 grid((a.total + 255) / 256), block(256);
  if (vec == 8) launch_pairs<DT, 8>(a, interleaved, st);
  else if (vec == 4) launch_pairs<DT, 4>(a, interleaved, st);
  else if (vec == 2) launch_pairs<DT, 2>(a, interleaved, st);
  else if (access == 8) hipLaunchKernelGGL((append_any_kernel<DT, 8>), grid, block, 0, st, a, interleaved);
  else hipLaunchKernelGGL((append_any_kernel<DT, 1>), grid, block, 0, st, a, interleaved);
}

}  // namespace

extern "C" int moba_hip_append_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                      const void* k, int64_t k_token_stride, int64_t k_head_stride,
                                      const void* v, int64_t v_token_stride, int64_t v_head_stride,
                                      int dtype, int N, int Hq, int Hkv, int D,
                                      const float* cos_sin, int max_pos, int rotary_dim,
                                      int interleaved, void* k_cache, void* v_cache, int num_pages,
                                      int page_size, const int* table, int B, int table_width,
                                      const int* token_seq, const int* token_pos,
                                      const int* offsets, void* q_out, int* status, void* stream) {
  if (dtype != 0 && dtype != 1) { moba_set_error("append_rotary: dtype must be 0 (bf16) or 1 (fp16)"); return MOBA_ERR_ARG; }
  if (N < 1 || Hq < 0 || Hkv < 1 || D < 1 || D > 256) { moba_set_error("append_rotary: nonempty N, Hkv and D in [1,256] required"); return MOBA_ERR_ARG; }
  if (rotary_dim < 2 || rotary_dim > D || rotary_dim % 2 || max_pos < 1) { moba_set_error("append_rotary: rotary_dim must be even, in [2, D], and the table nonempty"); return MOBA_ERR_ARG; }
  if (num_pages < 1 || page_size < 1 || B < 1 || table_width < 1) { moba_set_error("append_rotary: nonempty page pool and table required"); return MOBA_ERR_ARG; }
  if ((Hq > 0) != (q != nullptr) || (Hq > 0) != (q_out != nullptr)) { moba_set_error("append_rotary: q and q_out go together with Hq > 0"); return MOBA_ERR_ARG; }
  if ((int64_t)N * (Hq + 2ll * Hkv) * D >= 1ll << 31) { moba_set_error("append_rotary: more than 2^31 elements in one call"); return MOBA_ERR_ARG; }
  if (((uintptr_t)cos_sin & 15) != 0) { moba_set_error("append_rotary: the cos / sin table must be 16-byte aligned"); return MOBA_ERR_ARG; }
  AppendArgs a;
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.q_ts = q_token_stride; a.q_hs = q_head_stride;
  a.k_ts = k_token_stride; a.k_hs = k_head_stride;
  a.v_ts = v_token_stride; a.v_hs = v_head_stride;
  a.N = N; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.R = rotary_dim;
  a.cos_sin = (const float2*)cos_sin; a.max_pos = max_pos;
  a.kc = (uint16_t*)k_cache; a.vc = (uint16_t*)v_cache;
  a.num_pages = num_pages; a.P = page_size; a.by_page = fast_div(page_size);
  a.table = table; a.B = B; a.W = table_width;
  a.seq = token_seq; a.pos = token_pos; a.offsets = offsets;
  a.q_out = (uint16_t*)q_out; a.status = status;
  int access = row_access(k, a.k_ts, a.k_hs, D);
  access = std::min(access, row_access(v, a.v_ts, a.v_hs, D));
  access = std::min(access, row_access(k_cache, 0, 0, D));
  access = std::min(access, row_access(v_cache, 0, 0, D));
  if (Hq > 0) access = std::min({access, row_access(q, a.q_ts, a.q_hs, D), row_access(q_out, 0, 0, D)});
  if (dtype == 0) launch_append<0>(a, interleaved, access, (hipStream_t)stream);
  else launch_append<1>(a, interleaved, access, (hipStream_t)stream);
  return moba_launch_status("append_rotary");
}
