// gemm_mx.hip — MXFP4 products of many rows (prompts, large batches).
//
// A workgroup computes BM batch rows by BN outputs (BN / 2 gate/up pairs), its
// WM x WN waves a grid of equal parts of it. The k tiles of both operands go
// from global memory straight into LDS (no registers in between), in the order
// the lanes read them, through a ring of S stages; each wave waits for its own
// loads of a stage, then one barrier per stage publishes it, and the slot that
// the barrier retires is filled with the stage S - 1 ahead.
//
// Rows of several bf16 terms take one stage per term and k tile: all terms of a
// row add to the same f32 sums.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "mxfp4.h"
#include "mxfp4_dev.h"

namespace pgd {
namespace mx {
namespace {

// 64 lanes' 16 (4) bytes from global memory to consecutive places from the LDS
// address `to` on. Written in assembly (no output registers) because the
// compiler would otherwise let later LDS reads wait for these loads to land;
// the waits are the kernel's own.
__device__ __forceinline__ void dma16(const void* g, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(g) : "memory");
}
__device__ __forceinline__ void dma4(const void* g, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(g) : "memory");
}

template <bool FP4_, int BM_, int BN_, int WM_, int WN_, int S_, int OCC_ = 1>
struct Shape {
  static constexpr int OCC = OCC_;
  static constexpr bool FP4 = FP4_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, S = S_;
  static constexpr int W = WM * WN, MF = BM / WM / 16, NF = BN / WN / 16;
  // a stage's loads: 1 KiB of codes or terms each, and 256 B of weight scales
  // (the last may reach past the tile), NL and NS of them to a wave
  static constexpr int XI = BM / 16 * (FP4 ? 1 : 4), WI = BN / 16, WS = (BN + 63) / 64;
  static constexpr int NL = (XI + WI + W - 1) / W, NS = (WS + W - 1) / W, LOADS = NL + NS;
  static constexpr int X = XI * 1024, SC = X + WI * 1024, BYTES = SC + WS * 256;
  // activation scales: every fourth stage brings those of 4 k tiles, 16 B of a
  // row, into the other of two slots behind the ring
  static constexpr int XS = FP4 ? (BM + 63) / 64 : 0, NX = (XS + W - 1) / W;
  static constexpr int RING = S * BYTES, LDS = RING + 2 * XS * 1024;
  static_assert(S >= 2 && S <= (FP4 ? 5 : 8) && LDS * OCC <= 160 * 1024);
};

template <class T, int EPI>
__global__ __launch_bounds__(64 * T::W, T::W * T::OCC / 4) void gemm_kernel(Args a, int nmb, int nnb, int per_xcd, bool vec) {
  constexpr bool DUAL = EPI == MX_SWIGLU;
  constexpr int MF = T::MF, NF = T::NF, S = T::S;
  constexpr int NW = DUAL ? NF / 2 : NF;      // a wave's row tiles of outputs
  constexpr int NB = DUAL ? T::BN / 32 : T::BN / 16;  // the workgroup's
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  // XCD x takes the contiguous range [x per_xcd, (x + 1) per_xcd) of blocks
  // (workgroups are dealt to the 8 XCDs in turn), ordered in groups of 8 row
  // blocks, in a group output block by output block
  const int gi = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (gi >= nmb * nnb) return;
  const int g0 = gi / (8 * nnb) * 8, gw = min(8, nmb - g0), in = gi - g0 * nnb;
  const int m0 = (g0 + in % gw) * T::BM, nt0 = in / gw * NB;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i16 = lane & 15, q = lane >> 4;
  const int wm = wave / T::WN, wn = wave % T::WN;

  // An activation load takes 64 B (a k tile's codes, or a block's terms) of each
  // of 16 rows, four neighbouring lanes a row, so that they leave as one request.
  // The four 16 B parts of row i lie in LDS in the order 0..3 ^ i / 4: then the
  // 16 lanes that read one part of 16 rows at once meet no bank twice.
  const int lr = lane >> 2, lp = (lane & 3) ^ (lane >> 4);
  const int swz = i16 >> 2;
  // this wave's loads: sources without the k tile's offset (a wave with fewer
  // repeats the last: the same bytes to the same place)
  const uint8_t* src[T::NL];
#pragma unroll
  for (int k = 0; k < T::NL; ++k) {
    const int j = min(wave * T::NL + k, T::XI + T::WI - 1);
    if (j < T::XI) {
      if constexpr (T::FP4) {
        src[k] = a.p.codes + (size_t)min(m0 + j * 16 + lr, a.rows - 1) * a.p.ldc;
      } else {  // block j % 4 of 16 rows
        src[k] = reinterpret_cast<const uint8_t*>(a.x + (size_t)min(m0 + (j >> 2) * 16 + lr, a.rows - 1) * a.ldx) +
                 (j & 3) * 64 + lp * 16;
      }
    } else {  // row tile f of the stage: a wave's NF tiles, gate before up
      const int f = j - T::XI, w = f / NF, t = f % NF;
      const bool up = DUAL && t >= NW;
      const size_t nt = min(nt0 + w * NW + (up ? t - NW : t), a.nt - 1);
      src[k] = (up ? a.uc : a.wc) + nt * a.kt * 1024 + lane * 16;
    }
  }
  const uint8_t* ssrc[T::NS];
#pragma unroll
  for (int k = 0; k < T::NS; ++k) {
    const int f = min(wave * T::NS + k, T::WS - 1) * 4 + q, w = f / NF, t = f % NF;
    const bool up = DUAL && t >= NW;
    const size_t nt = min(nt0 + w * NW + (up ? t - NW : t), a.nt - 1);
    ssrc[k] = (up ? a.us : a.ws) + nt * a.kt * 64 + i16 * 4;
  }
  const uint8_t* xsrc[T::FP4 ? T::NX : 1];
  if constexpr (T::FP4) {
#pragma unroll
    for (int k = 0; k < T::NX; ++k)
      xsrc[k] = a.p.scales + (size_t)min(m0 + min(wave * T::NX + k, T::XS - 1) * 64 + lane, a.rows - 1) * a.p.lds;
  }
  // stage t: k tile t / terms, term t % terms; kt and term follow the loads
  const int terms = T::FP4 ? 1 : a.terms, steps = a.kt * terms;
  int lk = 0, lterm = 0;
  auto issue = [&](uint32_t st) {
    if constexpr (T::FP4) {  // (first: sync() may wait for these loads of a stage that it lets fly)
      if ((lk & 3) == 0) {
#pragma unroll
        for (int k = 0; k < T::NX; ++k)
          dma16(xsrc[k] + (size_t)lk * 4, lds0 + T::RING + (((lk >> 2) & 1) * T::XS + min(wave * T::NX + k, T::XS - 1)) * 1024);
      }
    }
#pragma unroll
    for (int k = 0; k < T::NL; ++k) {
      const int j = min(wave * T::NL + k, T::XI + T::WI - 1);
      const uint8_t* p;
      if (j < T::XI) {
        // (past a row's last block: that block again, its weights are zero)
        if constexpr (T::FP4) p = src[k] + (size_t)min(lk * 4 + lp, a.nblk - 1) * 16;
        else p = src[k] + (size_t)lk * (kMxTileK * 2) + lterm * a.term_stride * 2;
      } else {
        p = src[k] + (size_t)lk * 1024;
      }
      dma16(p, st + j * 1024);
    }
#pragma unroll
    for (int k = 0; k < T::NS; ++k)
      dma4(ssrc[k] + (size_t)lk * 64, st + T::SC + min(wave * T::NS + k, T::WS - 1) * 256);
    if (++lterm == terms) {
      lterm = 0;
      lk = min(lk + 1, a.kt - 1);  // (the loads past the last stage fill slots that nothing reads)
    }
  };

  f4 acc[NF][MF] = {};
  // LDS operands of a stage: its weights' codes and scales, and activations (FP4:
  // the whole k tile and its scales, else the quarter that matrix instruction j takes)
  struct WFrag {
    uint4 c[NF];
    uint32_t s[NF];
  };
  auto read_w = [&](WFrag& f, const uint8_t* st) {
    const uint8_t* ws = st + T::SC + wn * NF * 64 + lane;
    const uint8_t* wp = st + T::X + wn * NF * 1024 + lane * 16;
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      f.c[n] = *reinterpret_cast<const uint4*>(wp + n * 1024);
      f.s[n] = ws[n * 64];
    }
  };
  auto read_x = [&](uint4 (&x)[MF], const uint8_t* st, int j) {
    const uint8_t* xp = T::FP4 ? st + wm * MF * 1024 + i16 * 64 + (q ^ swz) * 16
                               : st + wm * MF * 4096 + q * 1024 + i16 * 64 + (j ^ swz) * 16;
#pragma unroll
    for (int m = 0; m < MF; ++m) x[m] = *reinterpret_cast<const uint4*>(xp + m * (T::FP4 ? 1024 : 4096));
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
  auto after = [&](uint32_t slot) { return slot + T::BYTES == S * T::BYTES ? 0 : slot + T::BYTES; };
  // All of the next stage's first operands are read under this stage's last
  // matrix instructions: the reads' latency and the barrier are hidden.
#pragma unroll
  for (int i = 0; i < S; ++i) issue(lds0 + i * T::BYTES);
  sync(std::integral_constant<int, S - 1>{});
  if constexpr (T::FP4) {
    struct Frag {
      WFrag w;
      uint4 x[MF];
      uint32_t s[MF];
    };
    auto read = [&](Frag& f, const uint8_t* st, int kt) {
      read_w(f.w, st);
      read_x(f.x, st, 0);
      const uint8_t* xs = smem + T::RING + ((kt >> 2) & 1) * (T::XS * 1024) + (wm * MF * 16 + i16) * 16 + (kt & 3) * 4 + q;
      const bool in_row = kt * 4 + q < a.nblk;  // (scale bytes past the row may be anything)
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        const uint32_t b = xs[m * 256];
        f.s[m] = in_row ? b : 127;
      }
    };
    auto step = [&](int t, const Frag& f, Frag& next) {
      sync(std::integral_constant<int, S - 2>{});
      issue(lds0 + here);
      here = after(here);
      read(next, smem + here, t + 1);
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[n][m] = mfma_fp4(f.w.c[n], f.w.s[n], f.x[m], f.s[m], acc[n][m]);
    };
    Frag f0, f1;
    read(f0, smem, 0);
    for (int t = 0;;) {
      step(t, f0, f1);
      if (++t == steps) break;
      step(t, f1, f0);
      if (++t == steps) break;
    }
  } else {
    auto mma = [&](const WFrag& w, const uint4 (&x)[MF], int j) {
      bf8 wf[NF];
#pragma unroll
      for (int n = 0; n < NF; ++n) wf[n] = fp4_bf16x8(reinterpret_cast<const uint32_t*>(&w.c[n])[j], e8m0_f32(w.s[n]));
#pragma unroll
      for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[n][m] = mfma_bf16(wf[n], __builtin_bit_cast(bf8, x[m]), acc[n][m]);
    };
    auto step = [&](const WFrag& w, WFrag& next, uint4 (&x0)[MF], uint4 (&x1)[MF]) {
      const uint8_t* st = smem + here;
      read_x(x1, st, 1);
      mma(w, x0, 0);
      read_x(x0, st, 2);
      mma(w, x1, 1);
      read_x(x1, st, 3);
      mma(w, x0, 2);
      sync(std::integral_constant<int, S - 2>{});
      issue(lds0 + here);
      here = after(here);
      read_w(next, smem + here);
      read_x(x0, smem + here, 0);
      mma(w, x1, 3);
    };
    WFrag w0, w1;
    uint4 x0[MF], x1[MF];
    read_w(w0, smem);
    read_x(x0, smem, 0);
    for (int t = 0;;) {
      step(w0, w1, x0, x1);
      if (++t == steps) break;
      step(w1, w0, x0, x1);
      if (++t == steps) break;
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load into LDS outlives the workgroup
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    const int r = m0 + (wm * MF + m) * 16 + i16;
    if (r >= a.rows) continue;
#pragma unroll
    for (int n = 0; n < NW; ++n) {
      const int o = (nt0 + wn * NW + n) * 16 + q * 4;
      if (o >= a.n_out) continue;
      f4 v = acc[n][m];
      if constexpr (DUAL) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = swiglu(v[e], acc[n + NW][m][e]);
      }
      store4<EPI>(a, vec, r, o, v);
    }
  }
}

template <class T, int EPI>
void launch(const Args& a, hipStream_t s) {
  const int nb = EPI == MX_SWIGLU ? T::BN / 32 : T::BN / 16;
  const long long nmb = (a.rows + (long long)T::BM - 1) / T::BM, nnb = (a.nt + nb - 1) / nb;
  PGD_CHECK(nmb * nnb < (1ll << 30), kErrShape, "too many outputs for one MXFP4 product");
  const int per_xcd = (int)((nmb * nnb + 7) / 8);
  PGD_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm_kernel<T, EPI>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS));
  hipLaunchKernelGGL((gemm_kernel<T, EPI>), dim3(per_xcd * 8), dim3(64 * T::W), T::LDS, s, a, (int)nmb, (int)nnb, per_xcd,
                     rows_vec(a.o));
  PGD_HIP(hipGetLastError());
}

template <class T>
void launch_epi(const Args& a, hipStream_t s) {
  if (a.uc) launch<T, MX_SWIGLU>(a, s);
  else if (a.o.res) launch<T, MX_RES>(a, s);
  else launch<T, MX_STORE>(a, s);
}

}  // namespace

void run_many(const Args& a, hipStream_t s) {
  if (a.p.codes) launch_epi<Shape<true, 256, 256, 2, 4, 3>>(a, s);
  else launch_epi<Shape<false, 128, 256, 2, 4, 3>>(a, s);
}

}  // namespace mx
}  // namespace pgd
