// mxfp4.h — MXFP4 (OCP microscaled 4-bit floating point) operands: the public
// row-major planes, the device layout of matrices, and the launchers.
//
// A block is 32 consecutive elements of a row: 4-bit codes (sign, 2 exponent
// and 1 mantissa bits: 0 .5 1 1.5 2 3 4 6) and one scale byte s that stands for
// 2^(s - 127); s = 255 makes the block NaN.
//
// Planes (activations, and what a matrix is made of): codes [rows][ldc bytes],
// element 2 i of a row in the low nibble of byte i, and scales [rows][lds bytes].
//
// Matrices: tiles of 16 rows by 128 columns. Lane l of a wave owns row l % 16 and
// block l / 16 of a tile, which is what one lane feeds the 16x16x128 scaled matrix
// instruction: 16 B of codes. Four row tiles and their scales lie together as one
// step of [row tile / 4][k tile]: codes [4][64 lanes][16 B], then scales [64 lanes]
// [4 B], a lane's four bytes one register of which the instruction picks one. So
// 64 rows stream through memory as one run of 4352 B steps. Rows and columns of the
// last tiles past the matrix are zeros.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "quant.h"

namespace pgd {

enum XType : int { X_F32 = 0, X_F16 = 1, X_BF16 = 2 };
inline int xtype_bytes(int t) { return t == X_F32 ? 4 : 2; }

constexpr int kMxBlock = 32, kMxTileN = 16, kMxTileK = 128;

inline int mx_row_tiles(int n) { return (n + kMxTileN - 1) / kMxTileN; }
inline int mx_k_tiles(int k) { return (k + kMxTileK - 1) / kMxTileK; }
constexpr int kMxStep = 4352, kMxStepScales = 4096;
inline size_t mx_bytes(int n, int k) { return (size_t)((mx_row_tiles(n) + 3) / 4) * mx_k_tiles(k) * kMxStep; }
// codes of lane 0 of a tile, and the scale byte of lane `lane` of it
__host__ __device__ inline size_t mx_code_off(int row_tile, int k_tile, int kt) {
  return ((size_t)(row_tile >> 2) * kt + k_tile) * kMxStep + (row_tile & 3) * 1024;
}
__host__ __device__ inline size_t mx_scale_off(int row_tile, int k_tile, int kt, int lane) {
  return ((size_t)(row_tile >> 2) * kt + k_tile) * kMxStep + kMxStepScales + lane * 4 + (row_tile & 3);
}

// Row-major planes on the device.
struct MxPlanes {
  const uint8_t* codes;
  int ldc;  // bytes, a multiple of 16
  const uint8_t* scales;
  int lds;  // bytes, a multiple of 16 (upload: any)
};

// Rows of x (XType, stride ldx elements) to planes; values (nullable, row
// stride ldv) receives what the codes stand for.
void mx_quantize(const void* x, int type, int ldx, int rows, int k, uint8_t* codes, int ldc, uint8_t* scales, int lds,
                 float* values, int ldv, hipStream_t s);
// planes of n_out rows into the planes of an allocated FMT_MXFP4 matrix
void mx_tile(QMat& m, const MxPlanes& p, hipStream_t s);
void mx_dequant(const QMat& m, int row0, int rows, float* out, hipStream_t s);

// What a product's epilogue does.
struct MxOut {
  float* y;
  int ldy;
  const float* res;  // nullable; may be y
  int ldres;
};
// y = W x (+ res), or with up: y = silu(W x) * (up x). x is rows of XType in
// device memory, or planes.
void mx_gemv(const QMat& w, const QMat* up, const void* x, int type, int ldx, int rows, const MxOut& o, hipStream_t s);
void mx_gemv_planes(const QMat& w, const QMat* up, const MxPlanes& x, int rows, const MxOut& o, hipStream_t s);

namespace mx {

constexpr int kMxDigitTile = 9216;  // 6 digits of 24 B a lane
// Workgroups of 256 threads of one launch, a multiple of 64: HIP takes grid sizes of less
// than 2^32 threads.
constexpr long long kMaxGroups = (1 << 24) - 64;

// How a launch holds its activation rows:
//   PLANES  p: the MXFP4 planes
//   TERMS   x: row r is the sum over t < terms of the bf16 rows
//           x[t * term_stride + r * ldx], of whole 128-column tiles
//   DIGITS  d, ds: six base-32 digits (mxfp4.hip), in tiles of 16 rows by 128
//           columns, [row tile][k tile]: kMxDigitTile bytes of e2m3 codes, 64 scales
//   ROWS    raw: rows of an XType with stride ldx, split by the launch itself
enum Kind : int { PLANES = 0, TERMS = 1, DIGITS = 2, ROWS = 3 };

// What the choice of a kernel goes by, and
struct Sizes {
  int n_out, nt, kt, nblk;  // outputs; row tiles, k tiles, 32-element blocks of a row
  int rows;
  bool pair;  // gate and up
  Kind kind;
  int terms;
};
// one product launch.
struct Args : Sizes {
  const uint8_t *w, *up;  // the matrix, and the up matrix (SwiGLU) or null
  MxPlanes p;
  const uint16_t* x;
  size_t ldx, term_stride;
  const void* raw;
  int raw_type;
  const uint8_t *d, *ds;
  MxOut o;
  // set by run_many: ranges of k tiles, and where their sums go
  int splits;
  float* part;
  size_t part_stride;
};

// A few rows (gemv_mx.hip; planes, terms or rows): in 64-row (of terms) chunks, its
// estimated microseconds; whether it can split that many rows of a type itself, and
// whether that beats splitting them first.
void run_few(const Args& a, hipStream_t s);
double few_us(const Sizes& a);
bool few_split_ok(int rows, int type);
bool few_split_pays(const Sizes& a, int type);
// Many rows (gemm_mx.hip; planes, terms or digits): the block shape and ranges of k tiles estimated
// fastest (more than one range only if scratch memory may be used).
struct Many {
  int shape, splits;
  int block_rows, block_outs;  // (outputs of both matrices for a pair)
  double us;
};
Many plan_many(const Sizes& a, bool scratch);
void run_many(const Args& a, const Many& m, hipStream_t s);

// What a product takes, from its sizes, type (an XType or X_PLANES), the stride of
// its rows in bytes (planes: the larger one) and whether scratch memory may be used.
struct Choice {
  Kind kind;
  bool prep;  // rows are split into scratch memory first
  bool few;   // run_few, or run_many by
  Many many;
};
constexpr int X_PLANES = 3;
Choice choose(int n_out, int n_in, bool pair, int type, long long stride, int rows, bool scratch);

}  // namespace mx
}  // namespace pgd
