// 8-bit KV pages: how a row of D values stands in the pool, and its conversions.
//
// A pool holds codes [num_pages][Hkv][P][Dp] (one byte each; Dp: D rounded up to
// 16) and scales [num_pages][Hkv][P] (fp32), for keys and for values.  A head's
// tokens lie one behind another, so that a pass over them reads whole cache
// lines at every D, and 16 scales of a page are one 64-byte piece.
//
//   a = max(max |x_d|, 2^-100),  s = a / top,  c_d = x_d top / a to the nearest
//   code (ties to the even one),  x_d ~ c_d s
//
// top is the largest code: 127 (format 0, int8) or 448 (format 1, the OCP 8-bit
// float e4m3).  A row that holds an infinity or a NaN has codes 0 and scale
// NaN: it reads back as NaN, and no code of it can harm a masked product.
#pragma once
#include "common.h"

namespace moba {

constexpr float kLeastMax = 0x1p-100f;  // 448 / a stays finite, rows of zeros divide by no zero
inline int code_width(int D) { return (D + 15) / 16 * 16; }
template <int FMT> constexpr float code_top() { return FMT == 0 ? 127.0f : 448.0f; }

// The factors of a row from the largest bit pattern of its |x| (an integer
// maximum, which keeps a NaN).  fold is a power of two that brings a into [1, 4),
// so that no product below overflows; inv is 1 / (a fold), rounded to nearest.
struct RowScale {
  float fold, a, inv, scale;
  bool finite;
};
template <int FMT> MOBA_DEV RowScale row_scale(uint32_t bits) {
  RowScale r;
  r.finite = bits < 0x7f800000u;
  const float a = fmaxf(__uint_as_float(r.finite ? bits : 0u), kLeastMax);
  const int e = min((int)(__float_as_uint(a) >> 23) - 127, 126);
  r.fold = __uint_as_float((uint32_t)(127 - e) << 23);
  r.a = a * r.fold;
  r.inv = 1.0f / r.a;
  r.scale = r.finite ? a / code_top<FMT>() : __uint_as_float(0x7fc00000u);
  return r;
}

// x top / a as the nearest fp32: a product by the reciprocal, and one correction
// by its residual, which the fused multiply-add has exactly.  x top is exact for a
// 16-bit x, and a quotient midway between two codes then comes out as just that.
template <int FMT> MOBA_DEV float to_code(float x, const RowScale& r) {
  const float p = x * r.fold * code_top<FMT>();
  const float q = p * r.inv;
  return fmaf(fmaf(-q, r.a, p), r.inv, q);
}

// Four quotients as four codes.  int8: adding 1.5 2^23 rounds to an integer whose low
// byte is the code.
template <int FMT> MOBA_DEV uint32_t codes4(float a, float b, float c, float d) {
  if constexpr (FMT == 0) {
    const uint32_t x = __float_as_uint(a + 12582912.0f), y = __float_as_uint(b + 12582912.0f);
    const uint32_t z = __float_as_uint(c + 12582912.0f), w = __float_as_uint(d + 12582912.0f);
    const uint32_t lo = __builtin_amdgcn_perm(y, x, 0x0c0c0400), hi = __builtin_amdgcn_perm(w, z, 0x04000c0c);
    return lo | hi;
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  }
}

// The numbers of four codes.
template <int FMT> MOBA_DEV void numbers4(uint32_t w, float (&x)[4]) {
  if constexpr (FMT == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = lo[0]; x[1] = lo[1]; x[2] = hi[0]; x[3] = hi[1];
  }
}

// The numbers of four codes in the 16-bit type, which has each of them exactly (at
// most 8 significant bits), as two packed words.
template <int FMT, int DT> MOBA_DEV void numbers4_16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == 1) {
    if constexpr (DT == 0) {
      lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
      hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
    } else {
      lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
      hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    }
  } else {
    float x[4];
    numbers4<0>(w, x);
    if constexpr (DT == 0) {  // the upper halves, as they are
      lo = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x07060302);
      hi = __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x07060302);
    } else {
      lo = pack2<1>(x[0], x[1]);
      hi = pack2<1>(x[2], x[3]);
    }
  }
}

// A pool and its page table, as every kernel of it has them.
struct QuantPool {
  uint8_t *k, *v;
  float *ks, *vs;
  int num_pages, P, Hkv, D, Dp;
  FastDiv by_page;
  const int* table;
  int B, W;
};

// Index of (token position, kv head) of a slot among the pool's rows; -1: none.
MOBA_DEV int64_t pool_row(const QuantPool& p, int slot, int pos, int kh) {
  if (slot < 0 || slot >= p.B || pos < 0) return -1;
  const uint32_t lp = div_by((uint32_t)pos, p.by_page);
  if (lp >= (uint32_t)p.W) return -1;
  const int page = p.table[(int64_t)slot * p.W + lp];
  if (page < 0 || page >= p.num_pages) return -1;
  return ((int64_t)page * p.Hkv + kh) * p.P + (pos - (int)(lp * p.by_page.d));
}

// 0, or an error with its message: what each entry checks of a pool.
int quant_pool_of(const char* what, int format, const void* k, const void* v, const float* ks,
                  const float* vs, int num_pages, int page_size, int Hkv, int D, const int* table,
                  int B, int W, QuantPool& p);

}  // namespace moba
