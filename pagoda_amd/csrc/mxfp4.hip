// mxfp4.hip — MXFP4 operands: quantization, matrix tiling, dequantization, the
// exact split of activation rows into bf16 terms, and the product front end.
#include <algorithm>
#include <mutex>

#include "common.h"
#include "gemv_impl.h"
#include "mxfp4.h"
#include "mxfp4_dev.h"

namespace pgd {

using namespace mx;

namespace {

// Eight consecutive elements of a row as f32.
template <int TYPE>
__device__ inline void load8(const void* x, size_t at, float (&v)[8]) {
  if constexpr (TYPE == X_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
    const float4 a = p[0], b = p[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == X_BF16) {
        v[2 * i] = __builtin_bit_cast(float, w[i] << 16);
        v[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
      } else {
        v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[i]);
        v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
      }
    }
  }
}

// Units (8 elements) of a row go to a power of two of threads, at most 256; the
// rest of a 256-thread workgroup takes further rows.
struct RowGrid {
  dim3 grid, block;
  RowGrid(int units, int rows) {
    int bx = 1;
    while (bx < units && bx < 256) bx *= 2;
    block = dim3(bx, 256 / bx);
    grid = dim3((units + bx - 1) / bx, std::min(((uint32_t)rows + block.y - 1) / block.y, 65535u));
  }
};

// A block's scale byte is the exponent of its largest magnitude less 2 (6 = 1.5
// 2^2 is the largest code), codes are rounded to nearest, ties to the even code,
// and saturate at 6: the conversion instruction's own rounding. Four threads
// share a block, so that a wave's loads and stores are runs of whole lines. Bound by
// HBM: each element is read once, its code and value written once. 2048 x 17408 f32 with
// values: 57 us, 5.35 TB/s; without them 28, 5.7 TB/s.
template <int TYPE>
__global__ __launch_bounds__(256) void quantize_kernel(const void* __restrict__ x, int ldx, uint32_t rows, int units,
                                                       uint8_t* __restrict__ codes, int ldc,
                                                       uint8_t* __restrict__ scales, int lds,
                                                       float* __restrict__ values, int ldv) {
  const int u = blockIdx.x * blockDim.x + threadIdx.x;
  if (u >= units) return;  // (units is a multiple of 4: a block's threads stay together)
  const uint32_t step = gridDim.y * blockDim.y;
  for (uint32_t r = blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += step) {
    float v[8];
    load8<TYPE>(x, (size_t)r * ldx + (size_t)u * 8, v);
    // magnitudes as bits: a NaN's exceed an infinity's, so nothing is lost to a maximum
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    const int e = (int)(top >> 23);
    const int sc = e == 255 ? 255 : max(e - 2, 0);
    const float scale = __builtin_bit_cast(float, (uint32_t)sc << 23);
    uint32_t c = 0;
    if (sc != 255) c = fp4_pack8(v, scale);
    *reinterpret_cast<uint32_t*>(codes + (size_t)r * ldc + (size_t)u * 4) = c;
    if ((u & 3) == 0) scales[(size_t)r * lds + (u >> 2)] = (uint8_t)sc;
    if (values) {
      float o[8];
      fp4_unpack8(c, scale, o);
      float* d = values + (size_t)r * ldv + (size_t)u * 8;
      reinterpret_cast<float4*>(d)[0] = make_float4(o[0], o[1], o[2], o[3]);
      reinterpret_cast<float4*>(d)[1] = make_float4(o[4], o[5], o[6], o[7]);
    }
  }
}

// One block (16 code bytes and its scale) per thread into its place in the tiles.
__global__ __launch_bounds__(256) void tile_kernel(MxPlanes p, int n_out, int nblk, int kt, uint8_t* __restrict__ w) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= nblk) return;
  const uint32_t step = gridDim.y * blockDim.y;
  for (int r = blockIdx.y * blockDim.y + threadIdx.y; r < n_out; r += step) {
    const int lane = (r & 15) + 16 * (b & 3);
    const uint4 c = *reinterpret_cast<const uint4*>(p.codes + (size_t)r * p.ldc + (size_t)b * 16);
    *reinterpret_cast<uint4*>(w + mx_code_off(r >> 4, b >> 2, kt) + lane * 16) = c;
    w[mx_scale_off(r >> 4, b >> 2, kt, lane)] = p.scales[(size_t)r * p.lds + b];
  }
}

__global__ __launch_bounds__(256) void dequant_kernel(const uint8_t* __restrict__ w, int row0, int rows, int units, int kt,
                                                      float* __restrict__ out) {
  const int u = blockIdx.x * blockDim.x + threadIdx.x;
  if (u >= units) return;
  const uint32_t step = gridDim.y * blockDim.y;
  for (int i = blockIdx.y * blockDim.y + threadIdx.y; i < rows; i += step) {
    const int r = row0 + i, b = u >> 2;
    const int lane = (r & 15) + 16 * (b & 3);
    const uint32_t c = *reinterpret_cast<const uint32_t*>(w + mx_code_off(r >> 4, b >> 2, kt) + lane * 16 + (u & 3) * 4);
    float o[8];
    fp4_unpack8(c, e8m0_f32(w[mx_scale_off(r >> 4, b >> 2, kt, lane)]), o);
    float* d = out + (size_t)i * units * 8 + (size_t)u * 8;
    reinterpret_cast<float4*>(d)[0] = make_float4(o[0], o[1], o[2], o[3]);
    reinterpret_cast<float4*>(d)[1] = make_float4(o[4], o[5], o[6], o[7]);
  }
}

// Rows as TERMS planes of bf16 terms (split_terms2). Columns [k, ldt) are zeros,
// which the last k tile reads. Bound by latency at the row counts that take it: 2 us
// for 5 f16 rows of 896.
template <int TYPE, int TERMS>
__global__ __launch_bounds__(256) void terms_kernel(const void* __restrict__ x, int ldx, uint32_t rows, int units,
                                                    uint16_t* __restrict__ out, int ldt, size_t term_stride) {
  const int u = blockIdx.x * blockDim.x + threadIdx.x;
  if (u * 8 >= ldt) return;
  const uint32_t step = gridDim.y * blockDim.y;
  for (uint32_t r = blockIdx.y * blockDim.y + threadIdx.y; r < rows; r += step) {
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (u < units) load8<TYPE>(x, (size_t)r * ldx + (size_t)u * 8, v);
    uint32_t t[4][TERMS];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float pair[2] = {v[2 * j], v[2 * j + 1]};
      split_terms2<TERMS>(pair, t[j]);
    }
#pragma unroll
    for (int i = 0; i < TERMS; ++i)
      *reinterpret_cast<uint4*>(out + i * term_stride + (size_t)r * ldt + (size_t)u * 8) =
          make_uint4(t[0][i], t[1][i], t[2][i], t[3][i]);
  }
}

// The 6-bit codes of three digits at once: 16 less the digit in bits 0..4, 10..14 and 20..24
// (others ignored) to a sign over a magnitude of 0..16 in bits 0..5, 10..15 and 20..25 (0 is -0).
__device__ __forceinline__ uint32_t digit_codes(uint32_t b) {
  const uint32_t minus = (b >> 4) & 0x100401, plus = minus ^ 0x100401;
  return (((b & 0xf03c0f) ^ plus * 15) + plus) | minus << 5;  // (below 16: 16 less the low bits)
}

// f32 rows in six base-32 digits. A block with largest magnitude below 2^(e - 126) (e
// the biased exponent, 26 at least) is held in steps of 2^(e - 155): 30 bits, so
// its values are exact to the last of their 24 where they are above 1/64 of the
// largest, and within 2^-30 of it elsewhere (f32 sums of its products keep 24).
// Digits -15..16 of that whole number, the top one from -16, are e2m3 codes (u / 8 is
// code u up to 16), digit i scaled by 2^(e - 128 - 5 i): half its worth, the products'
// kernel doubles its sums. Leading digits are up to 31/16 of their value (the others add up
// to less than 32^i 16/31 in digit i's unit), so halves stay below 2^128 whatever digits are
// still to come, wherever the magnitudes of the products add up to less. A tile of 16 rows by 128
// columns goes to 128 threads, half a block each (of lane l: block l / 16 of row l %
// 16). A block with an infinity or NaN is NaN. Rows and columns past the matrix are
// zeros. 333 rows of 5120: 8 us, latency (420 workgroups; one thread a block 1 us more);
// 868 rows of 3008: 11.5.
__global__ __launch_bounds__(256) void digits_kernel(const float* __restrict__ x, int ldx, int rows, int nblk, int kt,
                                                     uint32_t tiles, uint8_t* __restrict__ d,
                                                     uint8_t* __restrict__ ds) {
  const uint32_t tile = blockIdx.x * 2 + (threadIdx.x >> 7);
  if (tile >= tiles) return;
  const int lane = (threadIdx.x & 127) >> 1, half = threadIdx.x & 1;
  const uint32_t rt = tile / (uint32_t)kt, row = rt * 16 + (lane & 15);
  const int b = (int)(tile - rt * kt) * 4 + (lane >> 4);
  float v[2][8] = {};
  if (row < (uint32_t)rows && b < nblk) {
#pragma unroll
    for (int j = 0; j < 2; ++j) load8<X_F32>(x, (size_t)row * ldx + (size_t)b * kMxBlock + half * 16 + j * 8, v[j]);
  }
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __builtin_bit_cast(uint32_t, v[i >> 3][i & 7]) & 0x7fffffffu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1));
  const int e = max((int)(top >> 23), 26);
  uint32_t q[6][3] = {};  // [digit][dword]
  if (e != 255) {
    // (2^(155 - e) in two factors: it may pass the largest f32)
    const float up = __builtin_bit_cast(float, (uint32_t)(127 + (155 - e) / 2) << 23);
    const float up2 = __builtin_bit_cast(float, (uint32_t)(127 + (155 - e) - (155 - e) / 2) << 23);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      // (of the negative, whose digits are -16..15; 16 more in each of the lower five: their
      // bits are then 16 less the value's digits)
      const int n = 0x1084210 - __float2int_rn(v[i >> 3][i & 7] * up * up2);
      const int u = n >> 25;
      const uint32_t c5 = digit_codes((uint32_t)n), c4 = digit_codes((uint32_t)n >> 5);
#pragma unroll
      for (int k = 0; k < 6; ++k) {
        const uint32_t code = k ? (k & 1 ? c5 : c4) >> (k < 2 ? 20 : k < 4 ? 10 : 0) & 63
                                : (uint32_t)abs(u) | (u > 0 ? 32u : 0u);
        const int bit = 6 * i, w = bit >> 5, o = bit & 31;
        q[k][w] |= code << o;
        if (o > 26) q[k][w + 1] |= code >> (32 - o);
      }
    }
  }
  uint8_t* out = d + (size_t)tile * kMxDigitTile;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const uint32_t fourth = (uint32_t)__shfl_xor((int)q[k][0], 1);  // (the second half's first dword)
    if (half == 0) *reinterpret_cast<uint4*>(out + k * 1024 + lane * 16) = make_uint4(q[k][0], q[k][1], q[k][2], fourth);
    else *reinterpret_cast<uint2*>(out + 6144 + k * 512 + lane * 8) = make_uint2(q[k][1], q[k][2]);
  }
  if (half == 0) ds[(size_t)tile * 64 + lane] = (uint8_t)(e == 255 ? 255 : e - 1);
}

Sizes sizes_of(int n_out, int n_in, bool pair, int rows) {
  Sizes a{};
  a.n_out = n_out;
  a.nt = mx_row_tiles(n_out);
  a.kt = mx_k_tiles(n_in);
  a.nblk = n_in / kMxBlock;
  a.rows = rows;
  a.pair = pair;
  return a;
}

Args make_args(const QMat& w, const QMat* up, int rows, const MxOut& o) {
  Args a{sizes_of(w.n_out, w.n_in, up != nullptr, rows)};
  a.w = w.p0;
  a.up = up ? up->p0 : nullptr;
  a.o = o;
  return a;
}

long long digit_tiles(const Sizes& a) { return (long long)((a.rows - 1) / 16 + 1) * a.kt; }

int terms_of(int type) { return type == X_F32 ? 3 : type == X_F16 ? 2 : 1; }

// A captured graph would keep the address of scratch memory, which a later call
// may replace: captured launches use none.
bool scratch_allowed(hipStream_t s) { return !capturing(s); }

// Few or many rows' kernel, for rows of a kind.
Choice plan(const Sizes& a, size_t stride, bool scratch) {
  // (the many-row kernel's lanes hold offsets in 128 rows, and 16 row tiles of the matrix, in 32 bits)
  Choice c{a.kind, false, true, Many{0, 1, 0, 0, 1e30}};
  if (a.kind == DIGITS || stride < ((size_t)1 << 24)) c.many = plan_many(a, scratch), c.few = false;
  if (a.kind == DIGITS) return c;
  const double few = few_us(a);
  if (few <= c.many.us) c.few = true, c.many = Many{0, 1, 0, 0, few};
  return c;
}

void run(const Args& a, const Choice& c, hipStream_t s) {
  if (c.few) run_few(a, s);
  else run_many(a, c.many, s);
}

void check(const QMat& w, const QMat* up, int rows) {
  PGD_CHECK(w.fmt == FMT_MXFP4 && (!up || up->fmt == FMT_MXFP4), kErrFormat, "not an MXFP4 matrix");
  PGD_CHECK(!up || (up->n_out == w.n_out && up->n_in == w.n_in), kErrShape, "swiglu gate/up shapes differ");
  PGD_CHECK(rows >= 0, kErrShape, "gemv rows");
}

// The terms lie in the stream's scratch between the two launches. Held over
// both, so that no other host thread's call on the stream is queued between
// them or replaces the buffer.
std::mutex g_terms;

}  // namespace

void mx_quantize(const void* x, int type, int ldx, int rows, int k, uint8_t* codes, int ldc, uint8_t* scales, int lds,
                 float* values, int ldv, hipStream_t s) {
  if (rows == 0) return;
  const int units = k / 8;
  const RowGrid g(units, rows);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, g.grid, g.block, 0, s, x, ldx, rows, units, codes, ldc, scales, lds, values, ldv);
  };
  if (type == X_F32) go(quantize_kernel<X_F32>);
  else if (type == X_F16) go(quantize_kernel<X_F16>);
  else go(quantize_kernel<X_BF16>);
  PGD_HIP(hipGetLastError());
}

void mx_tile(QMat& m, const MxPlanes& p, hipStream_t s) {
  const int nblk = m.n_in / kMxBlock;
  const RowGrid g(nblk, m.n_out);
  hipLaunchKernelGGL(tile_kernel, g.grid, g.block, 0, s, p, m.n_out, nblk, mx_k_tiles(m.n_in), m.p0);
  PGD_HIP(hipGetLastError());
}

void mx_dequant(const QMat& m, int row0, int rows, float* out, hipStream_t s) {
  if (rows == 0) return;
  const int units = m.n_in / 8;
  const RowGrid g(units, rows);
  hipLaunchKernelGGL(dequant_kernel, g.grid, g.block, 0, s, m.p0, row0, rows, units, mx_k_tiles(m.n_in), out);
  PGD_HIP(hipGetLastError());
}

Choice mx::choose(int n_out, int n_in, bool pair, int type, long long stride, int rows, bool scratch) {
  Sizes a = sizes_of(n_out, n_in, pair, rows);
  if (type == X_PLANES) {
    a.kind = PLANES;
    return plan(a, stride, scratch);
  }
  a.terms = terms_of(type);
  a.kind = TERMS;
  if (type == X_BF16 && n_in % kMxTileK == 0) return plan(a, stride, scratch);  // the rows are their own term
  if (few_split_pays(a, type) || (!scratch && few_split_ok(rows, type))) return Choice{ROWS, false, true, Many{}};
  const size_t ldt = (size_t)a.kt * kMxTileK;
  Choice c = plan(a, ldt * 2, true);
  // (lanes hold offsets in two of the digits' row tiles in 32 bits, and two tiles go to a workgroup)
  if (type == X_F32 && rows > 16 && a.kt < (1 << 17) && digit_tiles(a) <= 2 * kMaxGroups) {
    // digits: 8.5 bytes of each value read and written instead of 10, and half the matrix
    // instructions' time (333 rows to a pair of 17408 x 5120: 193 us, as terms 256). 16
    // rows or fewer stay exact, so that a caller can have exact rows at any count; it costs
    // them time (5120 x 17408: 16 rows 30.8 us, 17 in digits 25.3; the pair: 57, 35).
    a.kind = DIGITS;
    const Choice d = plan(a, 0, true);
    if (d.many.us + 8.5 / 4.5e6 * rows * ldt < c.many.us + 10 / 4.5e6 * rows * ldt) c = d;
  }
  c.prep = true;
  return c;
}

void mx_gemv(const QMat& w, const QMat* up, const void* x, int type, int ldx, int rows, const MxOut& o, hipStream_t s) {
  check(w, up, rows);
  PGD_CHECK(type >= X_F32 && type <= X_BF16, kErrArg, "activations are f32 (0), f16 (1) or bf16 (2)");
  PGD_CHECK(ldx >= w.n_in && ldx % 8 == 0, kErrShape, "gemv ldx must be >= n_in and a multiple of 8");
  PGD_CHECK(reinterpret_cast<uintptr_t>(x) % 16 == 0, kErrArg, "MXFP4 activations must be 16-byte aligned");
  if (rows == 0) return;
  const bool scratch = scratch_allowed(s);
  const Choice c = choose(w.n_out, w.n_in, up, type, (long long)ldx * xtype_bytes(type), rows, scratch);
  Args a = make_args(w, up, rows, o);
  a.kind = c.kind;
  a.terms = terms_of(type);
  a.ldx = ldx;
  if (!c.prep) {  // TERMS: bf16 rows as they are, or ROWS
    a.x = static_cast<const uint16_t*>(x);
    a.raw = x;
    a.raw_type = type;
    run(a, c, s);
    return;
  }
  PGD_CHECK(scratch, kErrState,
            "splitting these MXFP4 activation rows needs scratch memory: under capture, at most 5 f32, 8 f16 or 4 bf16 "
            "rows, any bf16 rows of whole 128-column tiles, or MXFP4 rows");
  const int ldt = a.kt * kMxTileK;
  a.ldx = ldt;
  std::lock_guard<std::mutex> lock(g_terms);
  if (a.kind == DIGITS) {
    const long long tiles = digit_tiles(a);
    auto* d = static_cast<uint8_t*>(gemv::gemv_scratch(s, (size_t)tiles * (kMxDigitTile + 64), 8));
    auto* ds = d + (size_t)tiles * kMxDigitTile;
    a.d = d;
    a.ds = ds;
    hipLaunchKernelGGL(digits_kernel, dim3((unsigned)((tiles + 1) / 2)), dim3(256), 0, s, static_cast<const float*>(x), ldx,
                       rows, a.nblk, a.kt, (uint32_t)tiles, d, ds);
  } else {
    a.term_stride = (size_t)rows * ldt;
    auto* t = static_cast<uint16_t*>(gemv::gemv_scratch(s, a.terms * a.term_stride * sizeof(uint16_t), 8));
    a.x = t;
    const RowGrid g(ldt / 8, rows);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, g.grid, g.block, 0, s, x, ldx, rows, w.n_in / 8, t, ldt, a.term_stride);
    };
    if (type == X_F32) go(terms_kernel<X_F32, 3>);
    else if (type == X_F16) go(terms_kernel<X_F16, 2>);
    else go(terms_kernel<X_BF16, 1>);
  }
  PGD_HIP(hipGetLastError());
  run(a, c, s);
}

void mx_gemv_planes(const QMat& w, const QMat* up, const MxPlanes& x, int rows, const MxOut& o, hipStream_t s) {
  check(w, up, rows);
  if (rows == 0) return;
  Args a = make_args(w, up, rows, o);
  a.p = x;
  a.kind = PLANES;
  run(a, choose(w.n_out, w.n_in, up, X_PLANES, std::max(x.ldc, x.lds), rows, scratch_allowed(s)), s);
}

}  // namespace pgd
