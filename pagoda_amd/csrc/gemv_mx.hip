// gemv_mx.hip — MXFP4 products of a few rows.
//
// A workgroup of 8 waves owns NT row tiles of the matrix (of both matrices for
// the gate/up pair) and up to MT 16-row tiles of batch rows; its waves split
// the k tiles into 8 contiguous ranges, so a tile's weights (1 KiB of codes and
// 64 B of scales per k tile) are read once, in lane order, straight into the
// registers that feed the matrix instructions. The ranges' sums meet in LDS and
// are added in range order, so results do not depend on timing.
//
// Activation rows held as several bf16 terms take one matrix row per term and
// batch row (term t of row r is row t * rows + r), and the terms' sums are added
// at the end: a single f32 row costs one matrix instruction per 32 columns, not 3.
#include <algorithm>

#include "common.h"
#include "mxfp4.h"
#include "mxfp4_dev.h"

namespace pgd {
namespace mx {
namespace {

constexpr int kWaves = 8;

// One k tile of a batch row tile.
template <bool FP4>
struct XFrag;
template <>
struct XFrag<true> {
  uint4 c;
  uint32_t s;
};
template <>
struct XFrag<false> {
  uint4 c[4];
};

// A lane's batch row of each row tile. Lanes past the last row read that one
// again: column m of a product depends on row m alone, and theirs are dropped.
template <bool FP4>
struct XRow;
template <>
struct XRow<true> {
  const uint8_t *codes, *scales;
  XRow() = default;
  __device__ XRow(const Args& a, int m, int q) {
    m = min(m, a.rows - 1);
    codes = a.p.codes + (size_t)m * a.p.ldc;
    scales = a.p.scales + (size_t)m * a.p.lds;
  }
  // Blocks past the row's last: any codes (the weights are zero there), a scale of 1.
  __device__ XFrag<true> load(const Args& a, int kt, int q) const {
    const int b = kt * 4 + q, bc = min(b, a.nblk - 1);
    XFrag<true> f;
    f.c = *reinterpret_cast<const uint4*>(codes + (size_t)bc * 16);
    f.s = b < a.nblk ? scales[bc] : 127;
    return f;
  }
};
template <>
struct XRow<false> {
  const uint16_t* x;
  XRow() = default;
  __device__ XRow(const Args& a, int m, int q) {
    m = min(m, a.rows * a.terms - 1);
    const int t = m / a.rows;
    x = a.x + t * a.term_stride + (size_t)(m - t * a.rows) * a.ldx + q * 32;
  }
  __device__ XFrag<false> load(const Args& a, int kt, int q) const {
    XFrag<false> f;
    const uint4* p = reinterpret_cast<const uint4*>(x + (size_t)kt * kMxTileK);
#pragma unroll
    for (int j = 0; j < 4; ++j) f.c[j] = p[j];
    return f;
  }
};

template <int MT>
__device__ inline void mma(uint4 w, uint32_t ws, const XFrag<true> (&x)[MT], f4 (&acc)[MT]) {
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = mfma_fp4(w, ws, x[m].c, x[m].s, acc[m]);
}
// Matrix instruction j takes elements 8 j .. 8 j + 7 of each lane's block.
template <int MT>
__device__ inline void mma(uint4 w, uint32_t ws, const XFrag<false> (&x)[MT], f4 (&acc)[MT]) {
  const float s = e8m0_f32(ws);
  const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bf8 wf = fp4_bf16x8(c[j], s);
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = mfma_bf16(wf, __builtin_bit_cast(bf8, x[m].c[j]), acc[m]);
  }
}

template <bool FP4, int MT, int NT, int EPI>
__global__ __launch_bounds__(64 * kWaves) void few_kernel(Args a, int chunk, bool vec) {
  constexpr int NM = EPI == MX_SWIGLU ? 2 : 1;  // matrices
  __shared__ f4 part[kWaves][NM][NT][MT][64];
  // this workgroup's batch rows
  const int r0 = blockIdx.y * chunk;
  a.rows = min(chunk, a.rows - r0);
  if constexpr (FP4) {
    a.p.codes += (size_t)r0 * a.p.ldc;
    a.p.scales += (size_t)r0 * a.p.lds;
  } else {
    a.x += (size_t)r0 * a.ldx;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int q = lane >> 4;
  const int nt0 = blockIdx.x * NT;
  XRow<FP4> xr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = XRow<FP4>(a, m * 16 + (lane & 15), q);
  const uint8_t *wc[NM][NT], *ws[NM][NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const size_t tile = (size_t)min(nt0 + t, a.nt - 1) * a.kt;
    wc[0][t] = a.wc + tile * 1024 + lane * 16;
    ws[0][t] = a.ws + tile * 64 + lane;
    if constexpr (NM == 2) {
      wc[1][t] = a.uc + tile * 1024 + lane * 16;
      ws[1][t] = a.us + tile * 64 + lane;
    }
  }
  f4 acc[NM][NT][MT] = {};
  const int k1 = (int)((long long)(wave + 1) * a.kt / kWaves);
  for (int kt = (int)((long long)wave * a.kt / kWaves); kt < k1; ++kt) {
    XFrag<FP4> x[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = xr[m].load(a, kt, q);
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 w = *reinterpret_cast<const uint4*>(wc[i][t] + (size_t)kt * 1024);
        mma<MT>(w, ws[i][t][(size_t)kt * 64], x, acc[i][t]);
      }
  }
#pragma unroll
  for (int i = 0; i < NM; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) part[wave][i][t][m][lane] = acc[i][t][m];
  __syncthreads();
  // four outputs of one row per thread: ranges in order, terms in order
  const int terms = FP4 ? 1 : a.terms;
  for (int o = threadIdx.x; o < NT * 4 * a.rows; o += 64 * kWaves) {
    const int t = o / (4 * a.rows), rem = o - t * 4 * a.rows, nq = rem / a.rows, r = rem - nq * a.rows;
    f4 v[NM] = {};
    for (int term = 0; term < terms; ++term) {
      const int m = term * a.rows + r;
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
#pragma unroll
        for (int i = 0; i < NM; ++i) v[i] += part[w][i][t][m >> 4][nq * 16 + (m & 15)];
    }
    if constexpr (EPI == MX_SWIGLU) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[0][e] = swiglu(v[0][e], v[1][e]);
    }
    if (nt0 + t < a.nt) store4<EPI>(a, vec, r0 + r, (nt0 + t) * 16 + nq * 4, v[0]);
  }
}

template <bool FP4, int MT, int EPI>
void launch(const Args& a, int chunk, hipStream_t s) {
  constexpr int NT = EPI == MX_SWIGLU || MT > 2 ? 1 : 2;
  // (grid y is at most 65535: the rest goes to further launches)
  Args b = a;
  for (int r0 = 0; r0 < a.rows; r0 += chunk * 65535) {
    b.rows = (int)std::min<long long>(a.rows - r0, (long long)chunk * 65535);
    hipLaunchKernelGGL((few_kernel<FP4, MT, NT, EPI>), dim3((a.nt + NT - 1) / NT, (b.rows + chunk - 1) / chunk),
                       dim3(64 * kWaves), 0, s, b, chunk, rows_vec(a.o));
    PGD_HIP(hipGetLastError());
    if (b.rows == a.rows - r0) break;
    if constexpr (FP4) {
      b.p.codes += (size_t)b.rows * b.p.ldc;
      b.p.scales += (size_t)b.rows * b.p.lds;
    } else {
      b.x += (size_t)b.rows * b.ldx;
    }
    b.o.y += (size_t)b.rows * b.o.ldy;
    if (b.o.res) b.o.res += (size_t)b.rows * b.o.ldres;
  }
}

template <bool FP4, int MT>
void launch_epi(const Args& a, int chunk, hipStream_t s) {
  if (a.uc) launch<FP4, MT, MX_SWIGLU>(a, chunk, s);
  else if (a.o.res) launch<FP4, MT, MX_RES>(a, chunk, s);
  else launch<FP4, MT, MX_STORE>(a, chunk, s);
}

template <bool FP4>
void launch_rows(const Args& a, hipStream_t s) {
  const int terms = FP4 ? 1 : a.terms;
  const int chunk = std::min(a.rows, 64 / terms);
  switch ((chunk * terms + 15) / 16) {
    case 1: return launch_epi<FP4, 1>(a, chunk, s);
    case 2: return launch_epi<FP4, 2>(a, chunk, s);
    case 3: return launch_epi<FP4, 3>(a, chunk, s);
    default: return launch_epi<FP4, 4>(a, chunk, s);
  }
}

}  // namespace

void run_few(const Args& a, hipStream_t s) {
  if (a.p.codes) launch_rows<true>(a, s);
  else launch_rows<false>(a, s);
}

}  // namespace mx
}  // namespace pgd
