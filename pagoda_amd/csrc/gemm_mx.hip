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
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(g) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* g, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(g) : "memory", "m0");
}

template <bool FP4_, int BM_, int BN_, int WM_, int WN_, int S_>
struct Shape {
  static constexpr bool FP4 = FP4_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, S = S_;
  static constexpr int W = WM * WN, MF = BM / WM / 16, NF = BN / WN / 16;
  static constexpr int XI = BM / 16 * (FP4 ? 1 : 4), WI = BN / 16;  // 1 KiB loads of a stage
  static constexpr int SI = (FP4 ? BM / 64 : 0) + BN / 64;          // 256 B loads of scales
  static constexpr int NL = (XI + WI) / W;
  static constexpr int X = XI * 1024, SX = FP4 ? BM * 4 : 0;
  static constexpr int BYTES = X + WI * 1024 + SX + BN * 4;
  static_assert((XI + WI) % W == 0 && SI <= W && S >= 2, "every wave issues the same loads");
};

template <class T, int EPI>
__global__ __launch_bounds__(64 * T::W, T::W / 4) void gemm_kernel(Args a, int nmb, int nnb, int per_xcd, bool vec) {
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
  // this wave's loads: sources without the k tile's offset
  const uint8_t* src[T::NL];
#pragma unroll
  for (int k = 0; k < T::NL; ++k) {
    const int j = wave * T::NL + k;
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
  const int sj = wave % T::SI;  // (waves past the last load repeat one: the same bytes to the same place)
  const uint8_t* ssrc;
  constexpr int XS = T::FP4 ? T::BM / 64 : 0;
  if (sj < XS) {
    ssrc = a.p.scales + (size_t)min(m0 + sj * 64 + lane, a.rows - 1) * a.p.lds;
  } else {
    const int f = (sj - XS) * 4 + q, w = f / NF, t = f % NF;
    const bool up = DUAL && t >= NW;
    const size_t nt = min(nt0 + w * NW + (up ? t - NW : t), a.nt - 1);
    ssrc = (up ? a.us : a.ws) + nt * a.kt * 64 + i16 * 4;
  }
  // stage t: k tile t / terms, term t % terms; kt and term follow the loads
  const int terms = T::FP4 ? 1 : a.terms, steps = a.kt * terms;
  int lk = 0, lterm = 0;
  auto issue = [&](uint32_t st) {
#pragma unroll
    for (int k = 0; k < T::NL; ++k) {
      const int j = wave * T::NL + k;
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
    dma4(ssrc + (size_t)lk * (sj < XS ? 4 : 64), st + T::X + T::WI * 1024 + sj * 256);
    if (++lterm == terms) {
      lterm = 0;
      lk = min(lk + 1, a.kt - 1);  // (the loads past the last stage fill slots that nothing reads)
    }
  };

  f4 acc[NF][MF] = {};
  int ck = 0, cterm = 0;
  auto compute = [&](const uint8_t* st) {
    const uint8_t* ws = st + T::X + T::WI * 1024 + T::SX + wn * NF * 64 + lane;
    const uint8_t* wp = st + T::X + wn * NF * 1024 + lane * 16;
    uint4 w[NF];
    uint32_t sw[NF];
#pragma unroll
    for (int n = 0; n < NF; ++n) {
      w[n] = *reinterpret_cast<const uint4*>(wp + n * 1024);
      sw[n] = ws[n * 64];
    }
    if constexpr (T::FP4) {
      const uint8_t* xp = st + wm * MF * 1024 + i16 * 64 + (q ^ swz) * 16;
      const uint8_t* xs = st + T::X + T::WI * 1024 + (wm * MF * 16 + i16) * 4 + q;
      const bool in_row = ck * 4 + q < a.nblk;  // (scale bytes past the row may be anything)
#pragma unroll
      for (int m = 0; m < MF; ++m) {
        const uint4 x = *reinterpret_cast<const uint4*>(xp + m * 1024);
        const uint32_t sb = xs[m * 64], sx = in_row ? sb : 127;
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[n][m] = mfma_fp4(w[n], sw[n], x, sx, acc[n][m]);
      }
    } else {
      const uint8_t* xp = st + wm * MF * 4096 + q * 1024 + i16 * 64;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf8 wf[NF];
#pragma unroll
        for (int n = 0; n < NF; ++n) wf[n] = fp4_bf16x8(reinterpret_cast<const uint32_t*>(&w[n])[j], e8m0_f32(sw[n]));
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          const bf8 x = *reinterpret_cast<const bf8*>(xp + m * 4096 + (j ^ swz) * 16);
#pragma unroll
          for (int n = 0; n < NF; ++n) acc[n][m] = mfma_bf16(wf[n], x, acc[n][m]);
        }
      }
    }
    if (++cterm == terms) {
      cterm = 0;
      ++ck;
    }
  };
  // The stage has landed for every wave, and every wave has read the slot
  // that the next loads fill: S - 2 stages stay in flight.
  auto sync = [&] {
    constexpr int kFly = (S - 2) * (T::NL + 1);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((kFly & 15) | (7 << 4) | (kFly >> 4 << 14));  // vmcnt(kFly) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < S - 1; ++i) issue(lds0 + i * T::BYTES);
  uint32_t here = 0, next = (S - 1) * T::BYTES;  // the stage's slot, and the one that the loads fill
  for (int t = 0; t < steps; ++t) {
    sync();
    issue(lds0 + next);
    compute(smem + here);
    next = here;
    here = here + T::BYTES == S * T::BYTES ? 0 : here + T::BYTES;
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
  constexpr int lds = T::S * T::BYTES;
  static_assert(lds <= 160 * 1024);
  PGD_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&gemm_kernel<T, EPI>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds));
  hipLaunchKernelGGL((gemm_kernel<T, EPI>), dim3(per_xcd * 8), dim3(64 * T::W), lds, s, a, (int)nmb, (int)nnb, per_xcd,
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
