// kv8.h — the 8-bit paged KV cache: layout of a page, and the launches over it.
//
// A page holds kPage positions of every KV head:
//   codes   per KV head: K [hd / 64][4][16 positions][16 dims], then
//           V [hd / 64][4][16 dims][4][4 positions], one byte a code
//   bounds  per KV head: hd highest, then hd lowest key codes, int8
//   meta    per KV head: one u32 (Meta)
// padded to a multiple of 256 bytes. Both orders are those in which the lanes of a
// wave take matrix operands: lane l reads 16 bytes at 16 l of a 1 KiB run, of K
// position l % 16 and the dims 16 (l / 16).. of 64, of V the positions 4 (l / 16)..
// of the dims l % 16, 16 + l % 16, 32 + l % 16, 48 + l % 16 of 64.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pgd {
namespace kv8 {

constexpr int kPage = 16;             // positions of a page
constexpr int kMaxPages = 1 << 27;    // slots (page * 16 + place) are ints
constexpr int kExpMin = -126;         // smallest exponent of a (page, head)

enum Type { F32 = 0, F16 = 1, BF16 = 2 };

// A (page, head)'s u32: exponents of K and V plus 127, and the places whose K or V had a
// non-finite value (their codes are zero and they read as NaN).
struct Meta {
  __host__ __device__ static uint32_t pack(int ek, int ev, uint32_t nan) {
    return (uint32_t)(ek + 127) | (uint32_t)(ev + 127) << 8 | nan << 16;
  }
  __host__ __device__ static int ek(uint32_t m) { return (int)(m & 255u) - 127; }
  __host__ __device__ static int ev(uint32_t m) { return (int)(m >> 8 & 255u) - 127; }
  __host__ __device__ static uint32_t nan(uint32_t m) { return m >> 16; }
};

struct Layout {
  int kv_heads, hd;
  __host__ __device__ int head_bytes() const { return 2 * kPage * hd; }
  __host__ __device__ size_t bounds_at() const { return (size_t)kv_heads * head_bytes(); }
  __host__ __device__ size_t meta_at() const { return bounds_at() + (size_t)kv_heads * 2 * hd; }
  __host__ __device__ size_t page_bytes() const { return (meta_at() + (size_t)kv_heads * 4 + 255) & ~(size_t)255; }
};

// Offsets of a code among a head's K (or, plus 16 hd, V) codes.
__host__ __device__ inline int k_at(int place, int d) { return (d >> 4) * 256 + place * 16 + (d & 15); }
__host__ __device__ inline int v_at(int place, int d) {
  return (d >> 6) * 1024 + (place >> 2) * 256 + (d & 15) * 16 + (d >> 4 & 3) * 4 + (place & 3);
}

struct Pool {
  uint8_t* base;
  int n_pages;
  Layout at;
};

void append(const Pool& p, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, const int* slots, int rows,
            hipStream_t s);
void read(const Pool& p, const int* slots, int rows, float* k, int64_t ldk, float* v, int64_t ldv, hipStream_t s);

struct Tables {
  int block, nseq;
  const int *lens, *counts;
  int* tables;
  int max_blocks;
  const int* free_pages;
  int n_free;
  const int* taken;
  int rows;
  int *new_lens, *new_taken, *row_start, *seq_of_row, *pos_of_row, *slots, *status;
};
void tables(const Tables& t, hipStream_t s);

// The rows of an attention or selection call: sequence i owns rows
// [row_start[i], row_start[i + 1]), its latest, of a context of lens[i] positions.
struct Rows {
  int heads;
  const void* q;
  int64_t ldq;
  int type;
  int nseq;
  const int *row_start, *lens, *block_tables;
  int max_blocks, rows;
};
struct Out {
  void* out;
  int64_t ldo;
  const void* gate;  // nullable
  int64_t ldg;
};

// The most that a call of these or any smaller numbers needs.
size_t attn_ws_bytes(const Layout& at, int heads, int nseq, int max_blocks, int rows, int max_rows);
void attn(const Pool& p, const Rows& r, int max_rows, const Out& o, void* ws, hipStream_t s);

size_t select_ws_bytes(const Layout& at, int rows, int max_blocks);
void select(const Pool& p, const Rows& r, int top, int sinks, int recent, int* sel, int* count, void* ws, hipStream_t s);

// What a call needs, and the most that one of these or any smaller numbers of rows and pages needs.
size_t attn_sparse_ws_bytes(const Layout& at, int heads, int rows, int top);
size_t attn_sparse_ws_most(const Layout& at, int heads, int rows, int top);
void attn_sparse(const Pool& p, const Rows& r, int top, const int* sel, const int* count, const Out& o, void* ws,
                 hipStream_t s);

}  // namespace kv8
}  // namespace pgd
