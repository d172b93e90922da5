// gemv_mx.hip — MXFP4 products of a few rows.
//
// A workgroup owns NT row tiles of the matrix (of both matrices for the gate/up
// pair) and up to MT 16-row tiles of batch rows; its KW waves take the k tiles in
// turn, so a tile's weights (1 KiB of codes and 64 B of scales per k tile) are read
// once, in lane order, straight into the registers that feed the matrix
// instructions. The waves' sums meet in LDS and are added in wave order, so results
// do not depend on timing.
//
// Activation rows held as several bf16 terms take one matrix row per term and
// batch row (term t of row r is row t * rows + r), and the terms' sums are added
// at the end: a single f32 row costs one matrix instruction per 32 columns, not 3.
//
// Bound by HBM: the weights are read once, 4.25 bits each. Measured, weights from HBM (in
// brackets: from the last-level cache, where 2 to 5 matrices in turn fit it): a 2 x 17408 x
// 5120 pair and one f32 row 22.9 us, 4.15 TB/s (19.9; a large copy moves 4.85), 5120 x 17408
// and 8 MXFP4 rows 15.7 us, 3.05 TB/s (10.4), 151936 x 896 and 5 f16 rows 22.1 us, 3.4 TB/s
// with the launch that splits them (18.3). The first has 1088 workgroups, the second 160 of
// 8 waves: few bytes in flight. Past about 16 rows of terms every workgroup's reads of all
// activations from L2 weigh more than the weights (32 bf16 rows of 17408: 59 us in a
// graph, which takes no ranges of k tiles; 20 in blocks that share them through LDS with 6
// ranges, gemm_mx.hip).
#include <algorithm>

#include "common.h"
#include "mxfp4.h"
#include "mxfp4_dev.h"

namespace pgd {
namespace mx {
namespace {

// (KIND: PLANES, TERMS, or ROWS + XType for rows the launch splits itself: at most 16
// terms of rows, k any multiple of 32)

// One k tile of a batch row tile, as the matrix instructions take it.
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

// The activations of MT row tiles: load() asks for a k tile, frags() turns what
// came into operands. Lanes past the last row read that one again: column m of a
// product depends on row m alone, and theirs are dropped.
//
// Two neighbouring values of a row per lane, split into terms and put into the
// wave's own LDS as 16 rows of 256 B, the 16 B parts of row m in the order
// 0..15 ^ m: a lane's operand is one part of row lane % 16.
template <int KIND, int MT>
struct X {
  static_assert(KIND >= ROWS && MT == 1);
  static constexpr int TYPE = KIND - ROWS, T = TYPE == X_F32 ? 3 : TYPE == X_F16 ? 2 : 1, R = 16 / T;
  using Raw = uint32_t[R][TYPE == X_F32 ? 2 : 1];
  uint8_t* lds;
  __device__ X(const Args&, int, uint8_t* l) : lds(l) {}
  __device__ void load(const Args& a, int kt, int lane, Raw& f) const {
    const int k = kt * kMxTileK + lane * 2;
    const bool in = k < a.nblk * kMxBlock;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= a.rows) break;
      const size_t at = (size_t)r * a.ldx + k;
      if constexpr (TYPE == X_F32) {
        const uint2 v = in ? *reinterpret_cast<const uint2*>(static_cast<const float*>(a.raw) + at) : make_uint2(0, 0);
        f[r][0] = v.x;
        f[r][1] = v.y;
      } else {
        f[r][0] = in ? *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.raw) + at) : 0;
      }
    }
  }
  __device__ void frags(const Args& a, int, int lane, const Raw& f, XFrag<false> (&x)[1]) const {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r >= a.rows) break;
      float v[2];
      if constexpr (TYPE == X_F32) {
        v[0] = __builtin_bit_cast(float, f[r][0]);
        v[1] = __builtin_bit_cast(float, f[r][1]);
      } else if constexpr (TYPE == X_F16) {
        v[0] = (float)__builtin_bit_cast(_Float16, (uint16_t)f[r][0]);
        v[1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(f[r][0] >> 16));
      } else {
        v[0] = __builtin_bit_cast(float, f[r][0] << 16);
        v[1] = __builtin_bit_cast(float, f[r][0] & 0xffff0000u);
      }
      uint32_t t[T];
      split_terms2<T>(v, t);
#pragma unroll
      for (int i = 0; i < T; ++i) {
        const int m = i * a.rows + r;
        *reinterpret_cast<uint32_t*>(lds + m * 256 + (((lane >> 2) ^ m) & 15) * 16 + (lane & 3) * 4) = t[i];
      }
    }
    asm volatile("" ::: "memory");  // (one wave's LDS accesses run in order)
    const int m = lane & 15, q = lane >> 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[0].c[j] = *reinterpret_cast<const uint4*>(lds + m * 256 + ((q * 4 + j) ^ m) * 16);
    asm volatile("" ::: "memory");
  }
};
template <int MT>
struct X<PLANES, MT> {
  using Raw = XFrag<true>[MT];
  const uint8_t *codes[MT], *scales[MT];
  __device__ X(const Args& a, int lane, uint8_t*) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = min(m * 16 + (lane & 15), a.rows - 1);
      codes[m] = a.p.codes + (size_t)r * a.p.ldc;
      scales[m] = a.p.scales + (size_t)r * a.p.lds;
    }
  }
  // Blocks past the row's last: any codes (the weights are zero there), a scale of 1.
  __device__ void load(const Args& a, int kt, int lane, Raw& f) const {
    const int b = kt * 4 + (lane >> 4), bc = min(b, a.nblk - 1);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      f[m].c = *reinterpret_cast<const uint4*>(codes[m] + (size_t)bc * 16);
      const uint32_t s = scales[m][bc];
      f[m].s = b < a.nblk ? s : 127;
    }
  }
  __device__ void frags(const Args&, int, int, const Raw& f, XFrag<true> (&x)[MT]) const {
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = f[m];
  }
};
template <int MT>
struct X<TERMS, MT> {
  using Raw = XFrag<false>[MT];
  const uint16_t* x[MT];
  __device__ X(const Args& a, int lane, uint8_t*) {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = min(m * 16 + (lane & 15), a.rows * a.terms - 1), t = r / a.rows;
      x[m] = a.x + t * a.term_stride + (size_t)(r - t * a.rows) * a.ldx + (lane >> 4) * 32;
    }
  }
  __device__ void load(const Args&, int kt, int, Raw& f) const {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const uint4* p = reinterpret_cast<const uint4*>(x[m] + (size_t)kt * kMxTileK);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[m].c[j] = p[j];
    }
  }
  __device__ void frags(const Args&, int, int, const Raw& f, XFrag<false> (&x)[MT]) const {
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = f[m];
  }
};
// (the weights' scale is byte B of ws)
template <int B, int MT>
__device__ inline void mma(uint4 w, uint32_t ws, const XFrag<true> (&x)[MT], f4 (&acc)[MT]) {
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = mfma_fp4<B, 0>(w, ws, fp4_operand(x[m].c), x[m].s, acc[m]);
}
// Matrix instruction j takes elements 8 j .. 8 j + 7 of each lane's block.
template <int B, int MT>
__device__ inline void mma(uint4 w, uint32_t ws, const XFrag<false> (&x)[MT], f4 (&acc)[MT]) {
  const float s = e8m0_f32(ws >> (8 * B) & 255);
  const uint32_t c[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bf8 wf = fp4_bf16x8(c[j], s);
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = mfma_bf16(wf, __builtin_bit_cast(bf8, x[m].c[j]), acc[m]);
  }
}

template <int KIND, int MT, int NT, int EPI, int KW>
__global__ __launch_bounds__(64 * KW) void few_kernel(Args a, int chunk, bool vec) {
  constexpr int NM = EPI == MX_SWIGLU ? 2 : 1;  // matrices
  constexpr bool FP4 = KIND == PLANES;
  __shared__ union {
    f4 part[KW][NM][NT][MT][64];
    uint8_t x[KW][KIND >= ROWS ? 4096 : 16];
  } lds;
  auto& part = lds.part;
  // this workgroup's batch rows
  const int r0 = blockIdx.y * chunk;
  a.rows = min(chunk, a.rows - r0);
  if constexpr (FP4) {
    a.p.codes += (size_t)r0 * a.p.ldc;
    a.p.scales += (size_t)r0 * a.p.lds;
  } else if constexpr (KIND == TERMS) {
    a.x += (size_t)r0 * a.ldx;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups are dealt to the 8 XCDs in turn: those whose row tiles' scales lie
  // together (four tiles) follow each other on one XCD, and find them in its L2.
  constexpr int NG = 4 / NT;
  const int id = blockIdx.x >> 3;
  const int nt0 = (((id / NG) * 8 + (blockIdx.x & 7)) * NG + id % NG) * NT;
  if (nt0 >= a.nt) return;
  const X<KIND, MT> xs(a, lane, lds.x[wave]);
  // (the scales of NT row tiles are neighbouring bytes)
  const uint8_t *wc[NM][NT], *ws[NM];
  const size_t sat = mx_scale_off(nt0, 0, a.kt, lane);
  ws[0] = a.w + sat;
  if constexpr (NM == 2) ws[1] = a.up + sat;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const size_t at = mx_code_off(min(nt0 + t, a.nt - 1), 0, a.kt) + lane * 16;
    wc[0][t] = a.w + at;
    if constexpr (NM == 2) wc[1][t] = a.up + at;
  }
  f4 acc[NM][NT][MT] = {};
  // this wave's k tiles
  struct Tile {
    uint4 w[NM][NT];
    uint32_t s[NM];
    typename X<KIND, MT>::Raw x;
  };
  auto load = [&](Tile& t, int kt) {
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      const uint8_t* s = ws[i] + (size_t)kt * kMxStep;
      t.s[i] = NT == 2 ? *reinterpret_cast<const uint16_t*>(s) : *s;
#pragma unroll
      for (int n = 0; n < NT; ++n) t.w[i][n] = *reinterpret_cast<const uint4*>(wc[i][n] + (size_t)kt * kMxStep);
    }
    xs.load(a, kt, lane, t.x);
  };
  auto products = [&](const Tile& t, int kt) {
    XFrag<FP4> x[MT];
    xs.frags(a, kt, lane, t.x, x);
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      mma<0, MT>(t.w[i][0], t.s[i], x, acc[i][0]);
      if constexpr (NT == 2) mma<1, MT>(t.w[i][1], t.s[i], x, acc[i][1]);
    }
  };
  // (two k tiles' loads together measured 8% faster for one row of f32, 3% slower for planes)
  constexpr int U = MT == 1 && !FP4 ? 2 : 1;
  for (int kt = wave; kt < a.kt; kt += U * KW) {
    Tile t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(t[u], min(kt + u * KW, a.kt - 1));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u == 0 || kt + u * KW < a.kt) products(t[u], kt + u * KW);
  }
  if constexpr (KIND >= ROWS) __syncthreads();  // (the sums take the place of the activations)
#pragma unroll
  for (int i = 0; i < NM; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) part[wave][i][t][m][lane] = acc[i][t][m];
  __syncthreads();
  // four outputs of one row per thread: waves in order, terms in order
  const int terms = FP4 ? 1 : a.terms;
  for (int o = threadIdx.x; o < NT * 4 * a.rows; o += 64 * KW) {
    const int t = o / (4 * a.rows), rem = o - t * 4 * a.rows, nq = rem / a.rows, r = rem - nq * a.rows;
    f4 v[NM] = {};
    for (int term = 0; term < terms; ++term) {
      const int m = term * a.rows + r;
#pragma unroll
      for (int w = 0; w < KW; ++w)
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

template <int KIND, int MT, int EPI>
void launch(Args a, int chunk, hipStream_t s) {
  constexpr int NT = EPI == MX_SWIGLU || MT > 2 ? 1 : 2;
  // (a grid has kMaxGroups workgroups in x: the row tiles past them go to a launch of their
  // own; a multiple of 32 of them, so that steps and 16-byte stores stay whole)
  constexpr int kTiles = (int)(kMaxGroups / 32 * 32) * NT;
  if (a.nt > kTiles) {
    Args rest = a;
    rest.nt -= kTiles;
    rest.n_out -= kTiles * kMxTileN;
    rest.w += mx_code_off(kTiles, 0, a.kt);
    if (a.up) rest.up += mx_code_off(kTiles, 0, a.kt);
    rest.o.y += (size_t)kTiles * kMxTileN;
    if (a.o.res) rest.o.res += (size_t)kTiles * kMxTileN;
    launch<KIND, MT, EPI>(rest, chunk, s);
    a.nt = kTiles;
    a.n_out = kTiles * kMxTileN;
  }
  // (grid y is at most 65535: the rest goes to further launches)
  Args b = a;
  for (long long r0 = 0; r0 < a.rows; r0 += b.rows) {
    b.rows = (int)std::min<long long>(a.rows - r0, (long long)chunk * 65535);
    const dim3 grid((a.nt + 31) / 32 * (32 / NT), (b.rows + chunk - 1) / chunk);
    auto go = [&](auto kernel, int waves) { hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, s, b, chunk, rows_vec(a.o)); };
    // (one f32 row, 1088 pairs of row tiles: 20.4 us with 4 waves, 22.2 with 8; 8 MXFP4
    // rows, 160 workgroups: 16.2 with 4, 11.1 with 8)
    const bool wide = (long long)(a.nt + NT - 1) / NT * grid.y >= 512;
    if (wide) go(few_kernel<KIND, MT, NT, EPI, 4>, 4);
    else go(few_kernel<KIND, MT, NT, EPI, 8>, 8);
    PGD_HIP(hipGetLastError());
    if constexpr (KIND == PLANES) {
      b.p.codes += (size_t)b.rows * b.p.ldc;
      b.p.scales += (size_t)b.rows * b.p.lds;
    } else if constexpr (KIND == TERMS) {
      b.x += (size_t)b.rows * b.ldx;
    }
    b.o.y += (size_t)b.rows * b.o.ldy;
    if (b.o.res) b.o.res += (size_t)b.rows * b.o.ldres;
  }
}

template <int KIND, int MT>
void launch_epi(const Args& a, int chunk, hipStream_t s) {
  if (a.up) launch<KIND, MT, MX_SWIGLU>(a, chunk, s);
  else if (a.o.res) launch<KIND, MT, MX_RES>(a, chunk, s);
  else launch<KIND, MT, MX_STORE>(a, chunk, s);
}

template <int KIND>
void launch_rows(const Args& a, hipStream_t s) {
  const int terms = KIND == PLANES ? 1 : a.terms;
  const int chunk = std::min(a.rows, 64 / terms);
  switch ((chunk * terms + 15) / 16) {
    case 1: return launch_epi<KIND, 1>(a, chunk, s);
    case 2: return launch_epi<KIND, 2>(a, chunk, s);
    case 3: return launch_epi<KIND, 3>(a, chunk, s);
    default: return launch_epi<KIND, 4>(a, chunk, s);
  }
}

}  // namespace

// Splitting rows inside the launch saves another one and the scratch between them
// (2.6 us), and costs each workgroup about 0.05 + 0.03 (rows * terms) us per k tile
// of a wave: measured for 1, 2, 4, 5 and 8 rows over 12 matrices from 300 x 17408
// to 151936 x 896, where more than 5 workgroups per CU always lose.
bool few_split_ok(int rows, int type) { return rows <= (type == X_F32 ? 5 : type == X_F16 ? 8 : 4); }
bool few_split_pays(const Sizes& a, int type) {
  const int terms = type == X_F32 ? 3 : type == X_F16 ? 2 : 1;
  return few_split_ok(a.rows, type) && (a.pair ? a.nt : (a.nt + 1) / 2) <= 1280 &&
         (a.kt + 7) / 8 * (0.05 + 0.03 * a.rows * terms) <= 2.2;
}

// Microseconds of a launch; per 256 workgroups, their weight tiles and their
// activation tiles; per k tile, and row of terms of it (1..4 row tiles of rows).
// Fitted with the costs in gemm_mx.hip: 10 to 15% rms off, with weights from the last-level
// cache. From HBM a few rows take up to 1.5 times as long (one f32 row, 5120 x 17408: 19.3
// us, 12.3 here and 3 of the split); 8 f32 rows of a 17408 x 5120 pair take 73, 36 here.
double few_us(const Sizes& a) {
  static constexpr float kPlanes[4][6] = {{5.16f, 0.066f, 0.0257f, 0.00017f, 0.0005f, 0.0020f},
                                          {4.54f, 0.296f, 0.0188f, 0.0013f, 0.020f, 0.0024f},
                                          {4.04f, 0.384f, 0.0173f, 0.0018f, 0.0f, 0.0032f},
                                          {3.75f, 0.425f, 0.0333f, 0.0016f, 0.0f, 0.0029f}};
  static constexpr float kTerms[4][6] = {{4.28f, 0.223f, 0.0171f, 0.0039f, 0.019f, 0.0033f},
                                         {3.64f, 0.497f, 0.0179f, 0.0047f, 0.047f, 0.0038f},
                                         {3.15f, 0.142f, 0.0f, 0.0072f, 0.0f, 0.0053f},
                                         {3.45f, 0.400f, 0.0f, 0.0060f, 0.0f, 0.0050f}};
  const int terms = a.kind == PLANES ? 1 : a.terms, chunk = std::min(a.rows, 64 / terms), x = chunk * terms, mt = (x + 15) / 16;
  const int tiles = a.pair ? 1 : mt > 2 ? 1 : 2;
  const double wg = (double)((a.nt + tiles - 1) / tiles) * ((a.rows - 1) / chunk + 1) / 256.0;
  const float* c = a.kind == PLANES ? kPlanes[mt - 1] : kTerms[mt - 1];
  return c[0] + wg * (c[1] + a.kt * (c[2] * tiles * (a.pair ? 2 : 1) + c[3] * x)) + a.kt * (c[4] + c[5] * x);
}

void run_few(const Args& a, hipStream_t s) {
  if (a.kind == PLANES) return launch_rows<PLANES>(a, s);
  if (a.kind == TERMS) return launch_rows<TERMS>(a, s);
  switch (a.raw_type) {
    case X_F32: return launch_epi<ROWS + X_F32, 1>(a, a.rows, s);
    case X_F16: return launch_epi<ROWS + X_F16, 1>(a, a.rows, s);
    default: return launch_epi<ROWS + X_BF16, 1>(a, a.rows, s);
  }
}

}  // namespace mx
}  // namespace pgd
