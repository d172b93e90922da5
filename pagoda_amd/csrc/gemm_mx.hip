// gemm_mx.hip — MXFP4 products of many rows (prompts, large batches).
//
// A workgroup computes BM batch rows by BN outputs (BN / 2 gate/up pairs), its
// WM x WN waves a grid of equal parts of it. The k tiles of both operands go
// from global memory straight into LDS (no registers in between), in the order
// the lanes read them, through a ring of S stages; each wave waits for its own
// loads of a stage, then one barrier per stage publishes it, and the slot that
// the barrier retires is filled with the stage S - 1 ahead.
//
// y[r][n] = sum over 32-element blocks b of 2^(sx[r][b] + sw[n][b]) sum x w of the
// codes: the 4-bit instruction's own formula, for MXFP4 rows. Weights for bf16 rows
// are turned into bf16 (exactly) in registers, under the matrix instructions. Rows
// of several bf16 terms take one stage per term and k tile: all terms of a row add to
// the same f32 sums. Rows in digits (mxfp4.hip) take six matrix instructions of the
// 4-bit rate instead of three terms' twelve of the bf16 rate.
//
// Measured, inputs from HBM (17408 x 5120 unless given; MFMA: share of cycles the
// matrix units are busy):
//   4096 MXFP4 rows          252 us  2.90 PFLOP/s  MFMA 38%   blocks of 128 x 256
//   2048 MXFP4 rows, pair    235 us  3.10 PFLOP/s       42%   128 x 256
//   48 MXFP4 rows, pair       34 us  2.9 TB/s            14%  64 x 128
//   1999 bf16 rows of 6144 to 5120   117 us  1.08 PFLOP/s  61%   64 x 256
//   333 f32 rows, pair       193 us  digits: 0.62 PFLOP/s of the result, 57%   32 x 256
//   32 bf16 rows of 17408 to 5120    20 us  2.5 TB/s     21%  32 x 128, 6 ranges of k tiles
// Large MXFP4 products are bound by getting operands to the matrix units: a CU takes
// 43 B a clock from L2 into LDS at best (35 where rows give 64 B pieces) and needs 24
// KiB a stage of 512 clocks (585 to 700 of loads), and LDS serves a stage's 48 KiB of
// reads in 400. A CU's two blocks take about 2390 clocks for a stage of each, which is the
// sum of loads and matrix instructions and not the larger: they do not overlap as two
// blocks a CU should make them, and which wait keeps them apart is not known. Small ones
// are bound by the 2.5 to 3 TB/s that such loads reach from HBM: the loads alone take as
// long. bf16 rows run at nine tenths of what a large library product of bf16 reaches.
// Not taken, each at equal or longer times: weights straight into registers without
// LDS (equal for bf16 and digits; 5% slower for 4096 MXFP4 rows, 12 to 20% for pairs:
// the compiler's waits for them also wait for later LDS loads); longer rings (up to 8
// stages: the bytes in flight do not limit); blocks starting at different k tiles.
#include <algorithm>
#include <mutex>
#include <type_traits>
#include <utility>

#include "common.h"
#include "gemv_impl.h"
#include "mxfp4.h"
#include "mxfp4_dev.h"

namespace pgd {
namespace mx {
namespace {

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ const void* uniform(const void* p) {
  const uint64_t b = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<const void*>((uint64_t)uniform((uint32_t)(b >> 32)) << 32 | uniform((uint32_t)b));
}
// 64 lanes' 16 (4) bytes from base + off to consecutive places from the LDS
// address `to` on. Written in assembly (no output registers) because the
// compiler would otherwise let later LDS reads wait for these loads to land;
// the waits are the kernel's own. m0 is named as written: the compiler would
// else use a value it put there before (it warns that m0 is reserved: it keeps
// no variable there, which is what an m0 to be preserved would be).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(uniform(to)), "v"(off), "s"(uniform(base)) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* base, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(uniform(to)), "v"(off), "s"(uniform(base)) : "memory", "m0");
}
#pragma clang diagnostic pop

template <int KIND_, int BM_, int BN_, int WM_, int WN_, int S_, int OCC_ = 1>
struct Shape {
  static constexpr int KIND = KIND_;
  static constexpr bool FP4 = KIND == PLANES, DIG = KIND == DIGITS;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, S = S_, OCC = OCC_;
  static constexpr int W = WM * WN, MF = BM / WM / 16, NF = BN / WN / 16;
  // A wave's loads of a stage: NX of activations (XB bytes each, 4 or 16 a lane),
  // NL KiB of weight codes, NS times 256 B of weight scales (where there are
  // fewer than waves, several waves load the same bytes to the same place)
  static constexpr int X = BM / 16 * (FP4 ? 1024 : DIG ? kMxDigitTile : 4096), XB = DIG || X / 1024 % W == 0 ? 1024 : 256, XU = X / XB, NX = (XU + W - 1) / W;
  static constexpr int NL = BN / 16 / W, WS = BN / 64, NS = WS > W ? WS / W : 1, LOADS = NX + NL + NS + DIG;
  static constexpr int SC = X + BN * 64, DS = SC + BN * 4, BYTES = DS + (DIG ? BM * 4 : 0);
  // activation scales: every fourth stage brings those of 4 k tiles, 16 B of a
  // row, into the other of two slots behind the ring
  static constexpr int XS = FP4 ? (BM + 63) / 64 : 0, NXS = XS > W ? XS / W : 1;
  static constexpr int RING = S * BYTES, LDS = RING + 2 * XS * 1024;
  static_assert((!FP4 || MF == 1 || MF % 2 == 0) && (DIG || XU % W == 0) && BN / 16 % W == 0 && (WS <= W || WS % W == 0) && (XS <= W || XS % W == 0));
  static_assert(S >= 2 && S <= (FP4 ? 5 : 8) && LDS * OCC <= 160 * 1024 && (!DIG || BM <= 64));
};

// f(0), .., f(N - 1) with constant arguments
template <class F, int... I>
__device__ __forceinline__ void each(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
  each(f, std::make_integer_sequence<int, N>{});
}

template <class T, int EPI>
__global__ __launch_bounds__(64 * T::W, T::W * T::OCC / 4) void gemm_kernel(Args a, int nmb, int nnb, int per_xcd, bool vec) {
  constexpr bool DUAL = EPI == MX_SWIGLU || EPI == MX_PART2;
  constexpr int MF = T::MF, NF = T::NF, S = T::S;
  constexpr int NW = DUAL ? NF / 2 : NF;      // a wave's row tiles of outputs
  constexpr int NB = DUAL ? T::BN / 32 : T::BN / 16;  // the workgroup's
  static_assert(!DUAL || (NF % 2 == 0 && (T::NL == NF || NW % T::NL == 0)));
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const uint32_t lds0 = uniform((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem);
  // XCD x takes the contiguous range [x per_xcd, (x + 1) per_xcd) of blocks
  // (workgroups are dealt to the 8 XCDs in turn): range of k tiles by range, in
  // a range in groups of 8 row blocks, in a group output block by output block
  int gi = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (gi >= nmb * nnb * a.splits) return;
  const int split = uniform((uint32_t)(gi / (nmb * nnb)));  // (divisions leave the scalar unit)
  gi -= split * nmb * nnb;
  const int k0 = uniform((uint32_t)((long long)split * a.kt / a.splits)), k1 = uniform((uint32_t)((long long)(split + 1) * a.kt / a.splits));
  const int g0 = gi / (8 * nnb) * 8, gw = min(8, nmb - g0), in = gi - g0 * nnb;
  const int m0 = uniform((uint32_t)((g0 + in % gw) * T::BM)), nt0 = uniform((uint32_t)(in / gw * NB));
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i16 = lane & 15, q = lane >> 4;
  auto h = [](int g) { return (0x78 >> (2 * g)) & 3; };
  const int swz = h(i16 >> 2);
  const int wm = wave / T::WN, wn = wave % T::WN;

  // Where the bytes at LDS offset p of a stage come from, relative to the block's
  // first row and the k tile. A 16-row tile (a block of it, for bf16 terms) is 16
  // rows of 64 B, so that neighbouring lanes of a load leave as one request; the
  // four 16 B parts of row i lie in the order 0..3 ^ h(i / 4). An LDS read of 16 B a
  // lane takes lanes 0-3, 12-15, 20-27 at once (then the others of 32): with h = 0 2
  // 3 1 these meet no bank twice, whether the lanes' parts differ (codes: part l /
  // 16) or not (terms). Rows past the last are that row again, and are not stored.
  const int last = a.rows - 1 - m0;
  uint32_t xo[T::NX], cut[T::NX];
#pragma unroll
  for (int k = 0; k < T::NX; ++k) {
    const int p = min(wave * T::NX + k, T::XU - 1) * T::XB + lane * (T::XB / 64);
    const int i = (p >> 6) & 15, part = ((p >> 4) & 3) ^ h(i >> 2);
    if constexpr (T::DIG) {  // whole tiles, as they lie
      const int f = p / kMxDigitTile;
      xo[k] = (uint32_t)min(f, last >> 4) * (uint32_t)(a.kt * kMxDigitTile) + (p - f * kMxDigitTile);
    } else if constexpr (T::FP4) {
      xo[k] = (uint32_t)min((p >> 10) * 16 + i, last) * (uint32_t)a.p.ldc + part * 16 + (p & 15);
      // in the last k tile, blocks past the row's last are that one again (their weights are zero)
      cut[k] = max(part - ((a.nblk - 1) & 3), 0) * 16;
    } else {
      xo[k] = (uint32_t)min((p >> 12) * 16 + i, last) * (uint32_t)(a.ldx * 2) + ((p >> 10) & 3) * 64 + part * 16 + (p & 15);
    }
  }
  const uint8_t* xb = T::FP4   ? a.p.codes + (size_t)m0 * a.p.ldc
                      : T::DIG ? a.d + (size_t)(m0 >> 4) * a.kt * kMxDigitTile
                               : reinterpret_cast<const uint8_t*>(a.x + (size_t)m0 * a.ldx);
  // digits' scales: 64 B of each row tile
  const uint32_t dso = (uint32_t)min(q, last >> 4) * (uint32_t)(a.kt * 64) + i16 * 4;
  const uint8_t* dsb = T::DIG ? a.ds + ((size_t)(m0 >> 4) * a.kt + k0) * 64 : nullptr;
  // row tile f of the stage: a wave's NF tiles, gate before up
  auto tile_of = [&](int f, bool& up) {
    const int w = f / NF, t = f % NF;
    up = DUAL && t >= NW;
    return (size_t)min(nt0 + w * NW + (up ? t - NW : t), a.nt - 1);
  };
  const uint8_t *wb[T::NL], *sb[T::NS];
  const uint32_t wo = lane * 16;
#pragma unroll
  for (int k = 0; k < T::NL; ++k) {
    bool up;
    const size_t nt = tile_of(wave * T::NL + k, up);
    wb[k] = (up ? a.up : a.w) + mx_code_off((int)nt, k0, a.kt);
  }
  // weight scales, 4 row tiles a load: the gate's of the workgroup, then the up matrix's
#pragma unroll
  for (int k = 0; k < T::NS; ++k) {
    const int u = (wave * T::NS + k) % T::WS;
    const bool up = DUAL && u >= NB / 4;
    const size_t g = min(nt0 / 4 + (up ? u - NB / 4 : u), (a.nt - 1) / 4);
    sb[k] = (up ? a.up : a.w) + mx_scale_off((int)g * 4, k0, a.kt, 0);
  }
  const uint32_t wso = lane * 4;
  const uint8_t* xsb = a.p.scales + (T::FP4 ? (size_t)m0 * a.p.lds : 0);
  uint32_t xso[T::NXS];
#pragma unroll
  for (int k = 0; k < T::NXS; ++k)
    xso[k] = T::FP4 ? (uint32_t)min((wave * T::NXS + k) % max(T::XS, 1) * 64 + lane, last) * (uint32_t)a.p.lds : 0;

  // The loads' k tile and term. Past the last stage they repeat its k tile into
  // slots that nothing reads: every wave has the same number in flight.
  const int terms = T::KIND == TERMS ? a.terms : 1, steps = (k1 - k0) * terms;
  int lk = k0, lterm = 0;
  const size_t term_bytes = a.term_stride * 2;
  const uint8_t* xk = xb + (size_t)k0 * (T::FP4 ? 64 : T::DIG ? kMxDigitTile : 256);  // of k tile lk, term lterm
  bool first = true;
  auto issue = [&](uint32_t slot) {
    const uint32_t st = lds0 + slot;
    if constexpr (T::FP4) {  // (first: sync() may wait for these loads of a stage that it lets fly)
      if ((lk & 3) == 0 || first) {
        first = false;
#pragma unroll
        for (int k = 0; k < T::NXS; ++k)
          dma16(xsb + (size_t)(lk & ~3) * 4, xso[k],
                lds0 + T::RING + (((lk >> 2) & 1) * T::XS + (wave * T::NXS + k) % T::XS) * 1024);
      }
    }
    const bool end = lk == a.kt - 1;
#pragma unroll
    for (int k = 0; k < T::NX; ++k) {
      const uint32_t to = st + min(wave * T::NX + k, T::XU - 1) * T::XB;
      uint32_t off = xo[k];
      if constexpr (T::FP4) off -= end ? cut[k] : 0;
      if constexpr (T::XB == 1024) dma16(xk, off, to);
      else dma4(xk, off, to);
    }
#pragma unroll
    for (int k = 0; k < T::NL; ++k) dma16(wb[k], wo, st + T::X + (wave * T::NL + k) * 1024);
#pragma unroll
    for (int k = 0; k < T::NS; ++k) dma4(sb[k], wso, st + T::SC + (wave * T::NS + k) % T::WS * 256);
    if constexpr (T::DIG) {
      if (q < T::BM / 16) dma4(dsb, dso, st + T::DS);
    }
    // (no branches: the pointers stay in registers)
    const int more = T::KIND != TERMS ? lk + 1 < k1 : (lterm == terms - 1 && lk + 1 < k1);
    if constexpr (T::KIND != TERMS) {
      xk += more * (T::FP4 ? 64 : kMxDigitTile);
      if constexpr (T::DIG) dsb += more * 64;
    } else {
      const int wrap = lterm == terms - 1;
      xk += wrap ? more * 256 - (ptrdiff_t)term_bytes * (terms - 1) : (ptrdiff_t)term_bytes;
      lterm = wrap ? 0 : lterm + 1;
    }
    lk += more;
#pragma unroll
    for (int k = 0; k < T::NL; ++k) wb[k] += more * kMxStep;
#pragma unroll
    for (int k = 0; k < T::NS; ++k) sb[k] += more * kMxStep;
  };

  f4 acc[NF][MF] = {};
  // LDS operands of a stage: its weights' codes and scales, and of bf16 terms the
  // quarter that matrix instruction j takes
  // (scales: byte n % 4 of register n / 4 of a matrix's NW tiles; a wave with fewer
  // than 4 tiles shifts its own down)
  constexpr int NM = DUAL ? 2 : 1, SG = (NW + 3) / 4;
  static_assert(NB % 4 == 0 && (NW % 4 == 0 || 4 % NW == 0));
  struct WFrag {
    uint4 c[NF];
    uint32_t s[NM][SG];
  };
  auto read_w = [&](WFrag& f, uint32_t slot) {
    const uint8_t* ws = smem + slot + T::SC + (wn * NW >> 2) * 256 + lane * 4;
    const uint8_t* wp = smem + slot + T::X + wn * NF * 1024 + lane * 16;
#pragma unroll
    for (int n = 0; n < NF; ++n) f.c[n] = *reinterpret_cast<const uint4*>(wp + n * 1024);
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
      for (int g = 0; g < SG; ++g) {
        f.s[i][g] = *reinterpret_cast<const uint32_t*>(ws + (i * (NB / 4) + g) * 256);
        if constexpr (NW < 4) f.s[i][g] >>= 8 * (wn * NW & 3);
      }
  };
  auto ws_of = [](const WFrag& f, int n) { return f.s[n / NW][n % NW / 4]; };
  auto read_x = [&](uint4 (&x)[MF], uint32_t slot, int j) {
    const uint8_t* xp = smem + slot + wm * MF * 4096 + q * 1024 + i16 * 64 + (j ^ swz) * 16;
#pragma unroll
    for (int m = 0; m < MF; ++m) x[m] = *reinterpret_cast<const uint4*>(xp + m * 4096);
  };
  // A stage has landed for every wave, and every wave has read the slot that the
  // next loads fill. `fly` stages stay in flight.
  auto sync = [&](auto fly) {
    constexpr int kFly = decltype(fly)::value * T::LOADS;
    static_assert(kFly < 64);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((kFly & 15) | (7 << 4) | (kFly >> 4 << 14));  // vmcnt(kFly) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  uint32_t here = 0;  // the slot of the stage in use
  auto advance = [&] { here = here + T::BYTES == S * T::BYTES ? 0 : here + T::BYTES; };
  // Reads go out before the matrix instructions of what was read before: their
  // latency and the barrier's are hidden (the scheduler would put each next to its use).
  auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
#pragma unroll
  for (int i = 0; i < S; ++i) issue(i * T::BYTES);
  sync(std::integral_constant<int, S - 1>{});
  if constexpr (T::FP4) {
    // a stage in two halves of its row tiles
    constexpr int H = MF > 1 ? MF / 2 : 1;
    struct Half {
      uint4 x[H];
      uint32_t s[H];
    };
    auto read_half = [&](Half& f, int half, int kt) {
      const uint8_t* xp = smem + here + (wm * MF + half * H) * 1024 + i16 * 64 + (q ^ swz) * 16;
      const uint8_t* xs = smem + T::RING + ((kt >> 2) & 1) * (T::XS * 1024) + ((wm * MF + half * H) * 16 + i16) * 16 + (kt & 3) * 4 + q;
#pragma unroll
      for (int m = 0; m < H; ++m) {
        f.x[m] = *reinterpret_cast<const uint4*>(xp + m * 1024);
        f.s[m] = xs[m * 256];
      }
    };
    auto mma = [&](const WFrag& w, Half& f, int half, int kt) {
      if (kt == a.kt - 1 && kt * 4 + q >= a.nblk) {  // (scale bytes past the row may be anything)
#pragma unroll
        for (int m = 0; m < H; ++m) f.s[m] = 127;
      }
#pragma unroll
      for (int m = 0; m < H; ++m)
        each<NF>([&](auto n) {
          f4& c = acc[n][half * H + m];
          c = mfma_fp4<n % NW % 4, 0>(w.c[n], ws_of(w, n), fp4_operand(f.x[m]), f.s[m], c);
        });
      fence();
    };
    WFrag w0, w1;
    Half lo, hi;
    auto step = [&](int kt, const WFrag& w, WFrag& next) {
      if constexpr (MF > 1) {
        read_half(hi, 1, kt);
        fence();
        mma(w, lo, 0, kt);
      } else {
        hi = lo;
      }
      sync(std::integral_constant<int, S - 2>{});
      issue(here);
      advance();
      read_w(next, here);
      read_half(lo, 0, kt + 1);
      fence();
      mma(w, hi, MF > 1, kt);
    };
    read_w(w0, 0);
    read_half(lo, 0, k0);
    for (int t = 0;;) {
      step(k0 + t, w0, w1);
      if (++t == steps) break;
      step(k0 + t, w1, w0);
      if (++t == steps) break;
    }
  } else if constexpr (T::DIG) {
    // Three digits of a row tile at a time, the next three read under their products.
    struct Digits {
      i8v x[3];
    };
    auto read_digits = [&](Digits& f, int g) {
      const uint8_t* xp = smem + here + (wm * MF + (g >> 1)) * kMxDigitTile;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int d = (g & 1) * 3 + i;
        const uint4 lo = *reinterpret_cast<const uint4*>(xp + lane * 16 + d * 1024);
        const uint2 hi = *reinterpret_cast<const uint2*>(xp + lane * 8 + 6144 + d * 512);
        f.x[i] = (i8v){(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, 0, 0};
        // (joined into one read with the next digit's, hi would land outside its operand's registers)
        asm volatile("" ::: "memory");
      }
    };
    struct Stage {
      WFrag w;
      uint32_t s[MF];
    };
    auto read_stage = [&](Stage& f) {
      read_w(f.w, here);
#pragma unroll
      for (int m = 0; m < MF; ++m) f.s[m] = smem[here + T::DS + (wm * MF + m) * 64 + lane];
    };
    Digits even, odd;
    auto step = [&](const Stage& f, Stage& next) {
#pragma unroll
      for (int g = 0; g < 2 * MF; ++g) {
        Digits &now = g & 1 ? odd : even, &then = g & 1 ? even : odd;
        if (g + 1 < 2 * MF) {
          read_digits(then, g + 1);
        } else {
          sync(std::integral_constant<int, S - 2>{});
          issue(here);
          advance();
          read_stage(next);
          read_digits(then, 0);
        }
        fence();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const uint32_t s = f.s[g >> 1] - 5 * ((g & 1) * 3 + i);
          each<NF>([&](auto n) {
            acc[n][g >> 1] = mfma_fp4<n % NW % 4, 0, true>(f.w.c[n], ws_of(f.w, n), now.x[i], s, acc[n][g >> 1]);
          });
        }
        fence();
      }
    };
    Stage f0, f1;
    read_stage(f0);
    read_digits(even, 0);
    for (int t = 0;;) {
      step(f0, f1);
      if (++t == steps) break;
      step(f1, f0);
      if (++t == steps) break;
    }
  } else {
    auto decode = [&](bf8 (&wf)[NF], const WFrag& w, int j) {
#pragma unroll
      for (int n = 0; n < NF; ++n) wf[n] = fp4_bf16x8(reinterpret_cast<const uint32_t*>(&w.c[n])[j], e8m0_f32(ws_of(w, n) >> (8 * (n % NW % 4)) & 255));
    };
    auto mma = [&](const bf8 (&wf)[NF], const uint4 (&x)[MF]) {
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[n][m] = mfma_bf16(wf[n], __builtin_bit_cast(bf8, x[m]), acc[n][m]);
      // the next quarter's conversions in the shadows of these
#pragma unroll
      for (int i = 0; i < MF * NF; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, (4 * NF + MF * NF - 1) / (MF * NF), 0);
      }
      fence();
    };
    WFrag w;
    uint4 x0[MF], x1[MF];
    bf8 f0[NF], f1[NF];
    read_w(w, 0);
    read_x(x0, 0, 0);
    decode(f0, w, 0);
    for (int t = 0; t < steps; ++t) {
      read_x(x1, here, 1);
      fence();
      decode(f1, w, 1);
      mma(f0, x0);
      read_x(x0, here, 2);
      fence();
      decode(f0, w, 2);
      mma(f1, x1);
      read_x(x1, here, 3);
      fence();
      decode(f1, w, 3);
      mma(f0, x0);
      sync(std::integral_constant<int, S - 2>{});
      issue(here);
      advance();
      read_w(w, here);
      read_x(x0, here, 0);
      fence();
      mma(f1, x1);
      decode(f0, w, 0);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load into LDS outlives the workgroup
  if constexpr (T::DIG) {  // (digits are held at half their worth)
#pragma unroll
    for (int n = 0; n < NF; ++n)
#pragma unroll
      for (int m = 0; m < MF; ++m) acc[n][m] *= 2.0f;
  }
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    const uint32_t r = (uint32_t)m0 + (wm * MF + m) * 16 + i16;
    if (r >= (uint32_t)a.rows) continue;
#pragma unroll
    for (int n = 0; n < NW; ++n) {
      const int o = (nt0 + wn * NW + n) * 16 + q * 4;
      if (o >= a.n_out) continue;
      if constexpr (EPI == MX_PART || EPI == MX_PART2) {
        float* p = a.part + (size_t)split * a.part_stride + (size_t)r * (a.nt * 16) + o;
        *reinterpret_cast<f4*>(p) = acc[n][m];
        if constexpr (DUAL) *reinterpret_cast<f4*>(p + a.part_stride / 2) = acc[n + NW][m];
        continue;
      }
      f4 v = acc[n][m];
      if constexpr (EPI == MX_SWIGLU) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = swiglu(v[e], acc[n + NW][m][e]);
      }
      store4<EPI>(a, vec, r, o, v);
    }
  }
}

// Sums of the ranges in range order, then the epilogue: four outputs of a row per thread.
template <int EPI>
__global__ __launch_bounds__(256) void join_kernel(Args a, bool vec) {
  const int n = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (n >= a.n_out) return;
  for (uint32_t r = blockIdx.y; r < (uint32_t)a.rows; r += gridDim.y) {
    const float* p = a.part + (size_t)r * (a.nt * 16) + n;
    f4 v = {}, u = {};
#pragma unroll 4
    for (int i = 0; i < a.splits; ++i) {
      v += *reinterpret_cast<const f4*>(p + (size_t)i * a.part_stride);
      if constexpr (EPI == MX_SWIGLU) u += *reinterpret_cast<const f4*>(p + (size_t)i * a.part_stride + a.part_stride / 2);
    }
    if constexpr (EPI == MX_SWIGLU) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = swiglu(v[e], u[e]);
    }
    store4<EPI>(a, vec, r, n, v);
  }
}

template <class T, int EPI>
void launch_blocks(const Args& a, hipStream_t s) {
  const int nb = EPI == MX_SWIGLU || EPI == MX_PART2 ? T::BN / 32 : T::BN / 16;
  const long long nmb = (a.rows + (long long)T::BM - 1) / T::BM, nnb = (a.nt + nb - 1) / nb;
  PGD_CHECK(nmb * nnb * a.splits <= kMaxGroups, kErrShape, "too many outputs for one MXFP4 product");
  const int per_xcd = (int)((nmb * nnb * a.splits + 7) / 8);
  PGD_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm_kernel<T, EPI>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS));
  hipLaunchKernelGGL((gemm_kernel<T, EPI>), dim3(per_xcd * 8), dim3(64 * T::W), T::LDS, s, a, (int)nmb, (int)nnb,
                     per_xcd, rows_vec(a.o));
  PGD_HIP(hipGetLastError());
}

// The ranges' sums lie in the stream's scratch between the two launches. Held
// over both, so that no other host thread's call on the stream is queued
// between them or replaces the buffer.
std::mutex g_part;

template <class T>
void launch(Args a, int splits, hipStream_t s) {
  a.splits = splits;
  if (splits == 1) {
    if (a.up) launch_blocks<T, MX_SWIGLU>(a, s);
    else if (a.o.res) launch_blocks<T, MX_RES>(a, s);
    else launch_blocks<T, MX_STORE>(a, s);
    return;
  }
  std::lock_guard<std::mutex> lock(g_part);
  a.part_stride = (size_t)(a.up ? 2 : 1) * a.rows * a.nt * 16;
  a.part = static_cast<float*>(gemv::gemv_scratch(s, splits * a.part_stride * sizeof(float), 9));
  const dim3 grid((a.nt * 4 + 255) / 256, std::min(a.rows, 65535));
  auto join = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, rows_vec(a.o)); };
  if (a.up) {
    launch_blocks<T, MX_PART2>(a, s);
    join(join_kernel<MX_SWIGLU>);
  } else {
    launch_blocks<T, MX_PART>(a, s);
    if (a.o.res) join(join_kernel<MX_RES>);
    else join(join_kernel<MX_STORE>);
  }
  PGD_HIP(hipGetLastError());
}

// The shapes, largest first: wide ones read activations and weights fewer times from
// L2 and LDS per matrix instruction (4096 MXFP4 rows, 17408 x 5120: 32 x 128 blocks
// 606 us, 64 x 128 386, 128 x 128 333, 128 x 256 273); small ones give few rows blocks
// for all CUs (32 bf16 rows, 5120 x 17408, no ranges: 64 x 256 118, 64 x 128 77, 32 x
// 128 57; ranges of k tiles then bring it to 16). Two blocks share a CU, so that one
// computes while the other waits.
using P0 = Shape<PLANES, 128, 256, 1, 4, 3, 2>;
using P1 = Shape<PLANES, 128, 128, 2, 2, 4, 2>;
using P2 = Shape<PLANES, 64, 128, 1, 4, 4, 2>;
using P3 = Shape<PLANES, 32, 128, 1, 4, 5, 2>;
using T0 = Shape<TERMS, 64, 256, 1, 4, 2, 2>;
using T1 = Shape<TERMS, 64, 128, 1, 4, 3, 2>;
using T2 = Shape<TERMS, 32, 128, 1, 4, 4, 2>;
using D0 = Shape<DIGITS, 32, 256, 1, 4, 2, 2>;
using D1 = Shape<DIGITS, 32, 128, 2, 2, 3, 2>;

// Microseconds of a launch, of a stage and of the rest of a block where a CU runs
// two blocks and where it runs one, and of joining ranges (a launch, and each MB of
// their sums). Least squares over 11 matrices from 300 x 8192 to 151936 x 896 with
// 2..4000 rows, 1..24 ranges, weights from the last-level cache: 4 to 8% rms off. What they
// choose takes 1.008 times the fastest choice on the average of those, 1.19 at most. With
// inputs from HBM products take longer than estimated: 32 bf16 rows, 5120 x 17408, 20.1 us
// (16.5 here); 48 MXFP4 rows of a 17408 x 5120 pair 34 (22.9); 4096 to one matrix 252 (209);
// 333 f32 rows of the pair 193 with 8 us of digits (159).
struct Cost {
  int bm, bn;
  float launch, stage2, block2, stage1, block1, join, mb;
};
constexpr Cost kPlanes[] = {{128, 256, 6.45f, 0.995f, 3.90f, 0.630f, 2.13f, 1.66f, 0.269f},
                            {128, 128, 5.46f, 0.595f, 3.80f, 0.403f, 0.88f, 2.15f, 0.272f},
                            {64, 128, 4.93f, 0.396f, 2.17f, 0.293f, 0.07f, 2.52f, 0.299f},
                            {32, 128, 3.60f, 0.360f, 2.47f, 0.256f, 1.24f, 2.56f, 0.310f}};
constexpr Cost kTerms[] = {{64, 256, 6.22f, 1.311f, 1.13f, 0.813f, 0.00f, 1.85f, 0.282f},
                           {64, 128, 5.00f, 0.809f, 2.22f, 0.518f, 0.11f, 2.08f, 0.249f},
                           {32, 128, 3.63f, 0.512f, 2.19f, 0.382f, 0.61f, 2.38f, 0.281f}};
constexpr Cost kDigits[] = {{32, 256, 6.56f, 1.218f, 2.22f, 0.796f, 0.78f, 2.19f, 0.293f},
                            {32, 128, 5.73f, 0.757f, 2.58f, 0.526f, 1.24f, 2.14f, 0.278f}};

double cost_us(const Cost& c, const Sizes& a, int splits) {
  const int pair = a.pair ? 2 : 1;
  const long long blocks = (((long long)a.rows + c.bm - 1) / c.bm) * ((a.nt * 16ll * pair + c.bn - 1) / c.bn) * splits;
  if (blocks > kMaxGroups) return 1e30;
  const long long per_cu = (blocks + 255) / 256;
  const double stages = (a.kt + splits - 1) / splits * (a.kind == TERMS ? a.terms : 1);
  double us = c.launch + (double)(per_cu / 2) * (stages * c.stage2 + c.block2);
  if (per_cu % 2) us += stages * c.stage1 + c.block1;
  if (splits > 1) us += c.join + c.mb * 4e-6 * splits * a.rows * a.nt * 16.0 * pair;
  return us;
}

}  // namespace

Many plan_many(const Sizes& a, bool scratch) {
  Many best{0, 1, 0, 0, 1e30};
  const Cost* costs = a.kind == PLANES ? kPlanes : a.kind == TERMS ? kTerms : kDigits;
  const int shapes = a.kind == PLANES ? 4 : a.kind == TERMS ? 3 : 2;
  for (int i = 0; i < shapes; ++i)
    for (int splits : {1, 2, 3, 4, 6, 8, 10, 12, 16, 24}) {
      if (splits > 1 && (!scratch || splits * 2 > a.kt)) break;
      const double us = cost_us(costs[i], a, splits);
      if (us < best.us) best = Many{i, splits, costs[i].bm, costs[i].bn, us};
    }
  return best;
}

void run_many(const Args& a, const Many& m, hipStream_t s) {
  if (a.kind == PLANES) {
    switch (m.shape) {
      case 0: return launch<P0>(a, m.splits, s);
      case 1: return launch<P1>(a, m.splits, s);
      case 2: return launch<P2>(a, m.splits, s);
      default: return launch<P3>(a, m.splits, s);
    }
  }
  if (a.kind == DIGITS) return m.shape == 0 ? launch<D0>(a, m.splits, s) : launch<D1>(a, m.splits, s);
  switch (m.shape) {
    case 0: return launch<T0>(a, m.splits, s);
    case 1: return launch<T1>(a, m.splits, s);
    default: return launch<T2>(a, m.splits, s);
  }
}

}  // namespace mx
}  // namespace pgd
