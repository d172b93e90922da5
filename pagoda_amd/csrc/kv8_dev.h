// kv8_dev.h — device helpers shared by the kernels over the 8-bit KV cache.
#pragma once

#include <type_traits>

#include "common.h"
#include "kv8.h"

namespace pgd {
namespace kv8 {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// 2^e for e in [-126, 127], from its bits
__device__ inline float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

// Four values of magnitude up to 448 to e4m3 codes, to nearest, ties to even (the
// instruction's rounding; nothing here reaches its overflow).
__device__ inline uint32_t to_codes(float a, float b, float c, float d) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
__device__ inline f4 of_codes(uint32_t c) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  return f4{lo[0], lo[1], hi[0], hi[1]};
}

// The smallest exponent e >= -126 with top <= 448 * 2^e; 448 is 1.75 * 2^8.
__device__ inline int holds(float top) {
  const uint32_t b = __builtin_bit_cast(uint32_t, top);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e > kExpMin ? e : kExpMin;
}

// Eight elements of a row of type T as f32.
template <int T>
__device__ inline void load8(const void* p, int64_t i, float (&x)[8]) {
  if constexpr (T == F32) {
    const f4* q = reinterpret_cast<const f4*>(static_cast<const float*>(p) + i);
    const f4 a = q[0], b = q[1];
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = a[j], x[4 + j] = b[j];
  } else if constexpr (T == F16) {
    const h8 a = *reinterpret_cast<const h8*>(static_cast<const _Float16*>(p) + i);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = (float)a[j];
  } else {
    const u4 a = *reinterpret_cast<const u4*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = __builtin_bit_cast(float, (j & 1 ? a[j / 2] & 0xffff0000u : a[j / 2] << 16));
  }
}

// v combined with the values of the other lanes l ^ 16, l ^ 32, l ^ 48 (by two lane swaps,
// whose two results hold each lane's own value and its partner's).
template <class F>
__device__ inline float over_quads(float v, F f) {
  uint32_t b = __builtin_bit_cast(uint32_t, v);
  auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  v = f(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
  b = __builtin_bit_cast(uint32_t, v);
  r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return f(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ inline float quads_max(float v) {
  return over_quads(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline int quads_max(int v) {
  return __builtin_bit_cast(int, over_quads(__builtin_bit_cast(float, v), [](float a, float b) {
    return __builtin_bit_cast(float, max(__builtin_bit_cast(int, a), __builtin_bit_cast(int, b)));
  }));
}

// f over aligned groups of N lanes, the result in every lane, without LDS: within 16 lanes by exchanging
// neighbours, pairs, quads and halves, then by lane swaps.
template <int N, class T, class F>
__device__ inline T over_lanes(T v, F f) {
  auto other = [](T x, auto ctrl) {
    return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  auto swapped = [&](auto r) { return f(__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1])); };
  v = f(v, other(v, std::integral_constant<int, 0xb1>()));
  v = f(v, other(v, std::integral_constant<int, 0x4e>()));
  v = f(v, other(v, std::integral_constant<int, 0x141>()));
  if constexpr (N >= 16) v = f(v, other(v, std::integral_constant<int, 0x140>()));
  if constexpr (N >= 32) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    v = swapped(__builtin_amdgcn_permlane16_swap(b, b, false, false));
  }
  if constexpr (N >= 64) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    v = swapped(__builtin_amdgcn_permlane32_swap(b, b, false, false));
  }
  return v;
}
template <int N, class T>
__device__ inline T lanes_max(T v) {
  return over_lanes<N>(v, [](T a, T b) {
    if constexpr (std::is_same<T, float>::value) return fmaxf(a, b);
    else return max(a, b);
  });
}
template <int N, class T>
__device__ inline T lanes_min(T v) {
  return over_lanes<N>(v, [](T a, T b) { return min(a, b); });
}
__device__ inline float quads_sum(float v) {
  return over_quads(v, [](float a, float b) { return a + b; });
}

// Sums over the lanes before and with a lane, and over all lanes (identical in every lane).
template <int CTRL, int ROWS>
__device__ inline int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ inline int wave_scan(int v) {
  v = dpp_add<0x111, 0xf>(v);  // 1, 2, 4, 8 lanes of 16 up
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);  // lane 15 of a row to the next row, then lane 31 to the upper half
  return dpp_add<0x143, 0xc>(v);
}
template <int CTRL, int ROWS>
__device__ inline float dpp_addf(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
__device__ inline float wave_total(float v) {
  v = dpp_addf<0x111, 0xf>(v);
  v = dpp_addf<0x112, 0xf>(v);
  v = dpp_addf<0x114, 0xf>(v);
  v = dpp_addf<0x118, 0xf>(v);
  v = dpp_addf<0x142, 0xa>(v);
  v = dpp_addf<0x143, 0xc>(v);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// The sequence that owns a row (-1: none), with all that a row's context needs in one round of loads.
struct RowSeq {
  int seq, end, len;
  // positions that the row sees
  __device__ int seen(int row) const {
    return (int)max((long long)len - (end - 1 - row), 0ll);
  }
};
__device__ inline RowSeq row_seq(const Rows& r, int row) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < r.nseq; base += 64) {
    const int i = base + lane;
    int from = 0, end = 0, len = 0;
    if (i < r.nseq) from = r.row_start[i], end = r.row_start[i + 1], len = r.lens[i];
    const uint64_t hit = __ballot(i < r.nseq && from <= row && row < end);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      return RowSeq{base + src, min(__builtin_amdgcn_readlane(end, src), r.rows), __builtin_amdgcn_readlane(len, src)};
    }
  }
  return RowSeq{-1, 0, 0};
}

}  // namespace kv8
}  // namespace pgd
