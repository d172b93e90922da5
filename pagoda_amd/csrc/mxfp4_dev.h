// mxfp4_dev.h — device pieces of the MXFP4 kernels: 4-bit conversions, the two
// matrix instructions and the product epilogue.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mxfp4.h"

namespace pgd {
namespace mx {

using f4 = __attribute__((ext_vector_type(4))) float;
using bf2 = __attribute__((ext_vector_type(2))) __bf16;
using bf8 = __attribute__((ext_vector_type(8))) __bf16;
using f2v = __attribute__((ext_vector_type(2))) float;
using i8v = __attribute__((ext_vector_type(8))) int;

// 2^(s - 127), and for s = 255 an infinity, which the conversions below take as
// a NaN scale (byte 0 is a zero's bits: they read it as 2^-127).
__device__ inline float e8m0_f32(uint32_t s) { return __builtin_bit_cast(float, s << 23); }

// The conversion instructions read the exponent of the scale operand only.
__device__ inline uint32_t fp4_pack8(const float (&v)[8], float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
  return c;
}

__device__ inline void fp4_unpack8(uint32_t c, float scale, float (&o)[8]) {
  const f2v a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0);
  const f2v b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
  const f2v d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 2);
  const f2v e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 3);
  o[0] = a[0], o[1] = a[1], o[2] = b[0], o[3] = b[1], o[4] = d[0], o[5] = d[1], o[6] = e[0], o[7] = e[1];
}

// Exact: a code has 2 significant bits, and bf16 has f32's exponents.
__device__ inline bf8 fp4_bf16x8(uint32_t c, float scale) {
  const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0);
  const bf2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
  const bf2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2);
  const bf2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
  return (bf8){a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// x = t0 + t1 + t2 exactly: each term is the truncation to bf16 (8 significant
// bits) of what is left, so 3 terms hold the 24 bits of an f32, 2 the 11 of an
// f16 (but for bits below 2^-133, the smallest bf16 number). An infinity or NaN is its first term alone (a NaN stays one: its bits
// below bf16 are or-ed in). Two values, the terms packed low first.
template <int TERMS>
__device__ inline void split_terms2(float (&v)[2], uint32_t (&t)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; ++i) {
    uint32_t h[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float& x = v[e];
      const uint32_t b = __builtin_bit_cast(uint32_t, x);
      uint32_t hi = b & 0xffff0000u;
      const bool fin = (b & 0x7f800000u) != 0x7f800000u;
      if (!fin && (b & 0x007fffffu)) hi |= 0x00400000u;  // a NaN
      if (i + 1 < TERMS) x = fin ? x - __builtin_bit_cast(float, hi) : 0.0f;
      h[e] = hi;
    }
    t[i] = (h[0] >> 16) | h[1];
  }
}

// D[16 weight rows n][16 batch rows m]: lane l holds n = 4 (l / 16) + 0..3 of
// m = l % 16. Lane l feeds row l % 16 of either side.
__device__ inline f4 mfma_bf16(bf8 w, bf8 x, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0); }
// 128 columns of fp4 codes, lane l block l / 16, with those blocks' scales in byte
// WB (XB) of ws (xs); the activations' codes fp4, or e2m3 in 24 bytes (X6).
template <int WB, int XB, bool X6 = false>
__device__ inline f4 mfma_fp4(uint4 w, uint32_t ws, i8v x, uint32_t xs, f4 c) {
  const i8v a = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, x, c, 4, X6 ? 2 : 4, WB, (int)ws, XB, (int)xs);
}
__device__ inline i8v fp4_operand(uint4 x) { return (i8v){(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0}; }

// (PART, PART2: sums of a range of k tiles, of one matrix or of the pair)
enum { MX_STORE = 0, MX_RES = 1, MX_SWIGLU = 2, MX_PART = 3, MX_PART2 = 4 };

// silu(g) * u in f32: expf's error (an ulp or so) is that of the f32 products' sums
__device__ inline float swiglu(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// Four outputs n..n+3 of batch row r. vec: every row of y (and res) starts at a
// 16-byte boundary.
template <int EPI>
__device__ inline void store4(const Args& a, bool vec, int r, int n, f4 v) {
  float* y = a.o.y + (size_t)r * a.o.ldy + n;
  const float* res = EPI == MX_RES ? a.o.res + (size_t)r * a.o.ldres + n : nullptr;
  if (vec && n + 4 <= a.n_out) {
    if constexpr (EPI == MX_RES) v += *reinterpret_cast<const f4*>(res);
    *reinterpret_cast<f4*>(y) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < a.n_out) y[i] = EPI == MX_RES ? res[i] + v[i] : v[i];
}

inline bool rows_vec(const MxOut& o) {
  auto ok = [](const float* p, int ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 4 == 0; };
  return ok(o.y, o.ldy) && (!o.res || ok(o.res, o.ldres));
}

}  // namespace mx
}  // namespace pgd
