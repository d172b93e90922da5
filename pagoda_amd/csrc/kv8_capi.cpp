// kv8_capi.cpp — C entry points of the 8-bit paged KV cache: argument checks, then the launches.
#include "../../include/pagoda_hip.h"

#include <algorithm>

#include "device.h"
#include "kv8.h"

using namespace pgd;
using namespace pgd::kv8;

namespace {

constexpr int kMaxSeqs = 1 << 24;
constexpr int64_t kBlocks = 1 << 24;  // workgroups of 256 threads below a grid's 2^32 threads

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

bool head_dim_ok(int hd) { return hd == 64 || hd == 128 || hd == 256; }

Pool pool_of(const void* pool, int n_pages, int kv_heads, int head_dim) {
  PGD_CHECK(pool, kErrArg, "null pool");
  PGD_CHECK(aligned(pool, 16), kErrArg, "the pool must be 16-byte aligned");
  PGD_CHECK(head_dim_ok(head_dim), kErrShape, "head_dim must be 64, 128 or 256");
  PGD_CHECK(kv_heads > 0 && kv_heads <= 1024, kErrShape, "kv_heads must be 1..1024");
  PGD_CHECK(n_pages > 0 && n_pages < kMaxPages, kErrShape, "n_pages must be 1..2^27 - 1");
  return Pool{static_cast<uint8_t*>(const_cast<void*>(pool)), n_pages, Layout{kv_heads, head_dim}};
}

void check_rows(const void* p, int64_t ld, int64_t width, int unit, const char* what) {
  PGD_CHECK(p, kErrArg, std::string("null ") + what);
  PGD_CHECK(aligned(p, 16), kErrArg, std::string(what) + " must be 16-byte aligned");
  PGD_CHECK(ld >= width && ld % unit == 0, kErrShape,
            std::string(what) + " stride must be at least the row and a multiple of " + std::to_string(unit));
}

void check_type(int type) { PGD_CHECK(type >= F32 && type <= BF16, kErrArg, "type must be 0 (f32), 1 (f16) or 2 (bf16)"); }

// Sizes of an attention or selection call, as their workspace depends on them.
void check_sizes(const Layout& at, int heads, int nseq, int max_blocks, int rows) {
  PGD_CHECK(heads > 0 && heads % at.kv_heads == 0, kErrShape, "heads must be a multiple of kv_heads");
  PGD_CHECK(nseq >= 0 && rows >= 0, kErrArg, "nseq and rows must not be negative");
  PGD_CHECK(nseq <= kMaxSeqs, kErrShape, "nseq must be at most 2^24");
  PGD_CHECK(max_blocks > 0 && max_blocks <= 1 << 26, kErrShape, "max_blocks must be 1..2^26");
  const int64_t group = heads / at.kv_heads, tiles = rows * group / 16 + (nseq < rows ? nseq : rows);
  // (the join has a workgroup for four results of a row and head)
  PGD_CHECK((int64_t)rows * heads + 3 < kBlocks * 4 && tiles * at.kv_heads < kBlocks / 2, kErrShape,
            "more rows or sequences than one launch holds");
}

Rows rows_of(const Pool& p, int heads, const void* q, int ldq, int type, int nseq, const int* row_start,
             const int* lens, const int* block_tables, int max_blocks, int rows) {
  check_type(type);
  check_sizes(p.at, heads, nseq, max_blocks, rows);
  if (rows > 0 && nseq > 0) {
    check_rows(q, ldq, (int64_t)heads * p.at.hd, 8, "q");
    PGD_CHECK(row_start && lens && block_tables, kErrArg, "null argument");
  }
  return Rows{heads, q, ldq, type, nseq, row_start, lens, block_tables, max_blocks, rows};
}

Out out_of(const Rows& r, const Layout& at, void* out, int ldo, const void* gate, int ldg) {
  check_rows(out, ldo, (int64_t)r.heads * at.hd, 8, "out");
  if (gate) check_rows(gate, ldg, (int64_t)r.heads * at.hd, 8, "gate");
  return Out{out, ldo, gate, ldg};
}

void check_ws(const void* ws, size_t have, size_t need) {
  if (need == 0) return;
  PGD_CHECK(ws, kErrArg, "null workspace");
  PGD_CHECK(aligned(ws, 16), kErrArg, "the workspace must be 16-byte aligned");
  PGD_CHECK(have >= need, kErrShape, "the workspace has " + std::to_string(have) + " bytes of " + std::to_string(need));
}

// Rows times KV heads times the tiles of a group: what the launches of a list count in.
void check_list(const Layout& at, int heads, int rows, int max_blocks, int top) {
  PGD_CHECK(top > 0 && top <= 1 << 20, kErrShape, "top must be 1..2^20");
  const int64_t units = (int64_t)rows * at.kv_heads;
  PGD_CHECK(units < kBlocks / 4 && units * ((max_blocks + 127) / 128) < kBlocks, kErrShape,
            "more rows and pages than one launch holds");
  PGD_CHECK(units * ((heads / at.kv_heads + 15) / 16) < kBlocks / 8, kErrShape, "more rows than one launch holds");
}

size_t sparse_ws(const Layout& at, int heads, int rows, int max_blocks, int top) {
  const size_t a = select_ws_bytes(at, rows, max_blocks), b = attn_sparse_ws_most(at, heads, rows, top);
  return a > b ? a : b;
}

// The workspace of sizes that a call would refuse is 0.
template <class F>
size_t bytes_or_zero(F&& f) {
  size_t n = 0;
  return guard([&] { n = f(); }) == kOk ? n : 0;
}

}  // namespace

extern "C" {

size_t pgd_kv8_page_bytes(int kv_heads, int head_dim) {
  return kv_heads > 0 && kv_heads <= 1024 && head_dim_ok(head_dim) ? Layout{kv_heads, head_dim}.page_bytes() : 0;
}

int pgd_kv_tables_dev(pgd_dev* dev, int block, int nseq, const int* lens, const int* counts, int* tables_io,
                      int max_blocks, const int* free_pages, int n_free, const int* taken, int rows, int* new_lens,
                      int* new_taken, int* row_start, int* seq_of_row, int* pos_of_row, int* slots, int* status) {
  return guard([&] {
    PGD_CHECK(dev, kErrArg, "null device");
    PGD_CHECK(block > 0 && max_blocks > 0 && nseq >= 0 && n_free >= 0 && rows >= 0, kErrArg, "bad sizes");
    PGD_CHECK(nseq <= kMaxSeqs && rows <= 1 << 30, kErrShape, "nseq must be at most 2^24 and rows at most 2^30");
    PGD_CHECK(taken && new_taken && row_start, kErrArg, "null argument");
    PGD_CHECK(nseq == 0 || (lens && counts && tables_io && new_lens && status), kErrArg, "null argument");
    PGD_CHECK(n_free == 0 || free_pages, kErrArg, "null free list");
    PGD_CHECK(rows == 0 || (seq_of_row && pos_of_row && slots), kErrArg, "null row maps");
    DeviceScope scope(dev);
    tables(Tables{block, nseq, lens, counts, tables_io, max_blocks, free_pages, n_free, taken, rows, new_lens, new_taken,
                  row_start, seq_of_row, pos_of_row, slots, status},
           dev->stream);
  });
}

int pgd_kv8_append_dev(pgd_dev* dev, void* pool, int n_pages, int kv_heads, int head_dim, const void* k, int ldk,
                       const void* v, int ldv, int type, const int* slots, int rows) {
  return guard([&] {
    PGD_CHECK(dev, kErrArg, "null device");
    const Pool p = pool_of(pool, n_pages, kv_heads, head_dim);
    check_type(type);
    PGD_CHECK(rows >= 0, kErrArg, "rows must not be negative");
    PGD_CHECK((int64_t)rows * kv_heads < kBlocks, kErrShape, "more rows than one launch holds");
    if (rows == 0) return;
    PGD_CHECK(slots, kErrArg, "null slots");
    check_rows(k, ldk, (int64_t)kv_heads * head_dim, 8, "k");
    check_rows(v, ldv, (int64_t)kv_heads * head_dim, 8, "v");
    DeviceScope scope(dev);
    append(p, k, ldk, v, ldv, type, slots, rows, dev->stream);
  });
}

int pgd_kv8_read_dev(pgd_dev* dev, const void* pool, int n_pages, int kv_heads, int head_dim, const int* slots,
                     int rows, float* k, int ldk, float* v, int ldv) {
  return guard([&] {
    PGD_CHECK(dev, kErrArg, "null device");
    const Pool p = pool_of(pool, n_pages, kv_heads, head_dim);
    PGD_CHECK(rows >= 0, kErrArg, "rows must not be negative");
    PGD_CHECK((int64_t)rows * kv_heads < kBlocks * 32, kErrShape, "more rows than one launch holds");
    if (rows == 0) return;
    PGD_CHECK(slots, kErrArg, "null slots");
    check_rows(k, ldk, (int64_t)kv_heads * head_dim, 4, "k");
    check_rows(v, ldv, (int64_t)kv_heads * head_dim, 4, "v");
    DeviceScope scope(dev);
    read(p, slots, rows, k, ldk, v, ldv, dev->stream);
  });
}

size_t pgd_attn_kv8_ws_bytes(int heads, int kv_heads, int head_dim, int nseq, int max_blocks, int rows) {
  return pgd_attn_kv8_rows_ws_bytes(heads, kv_heads, head_dim, nseq, max_blocks, rows, std::max(rows, 0));
}

size_t pgd_attn_kv8_rows_ws_bytes(int heads, int kv_heads, int head_dim, int nseq, int max_blocks, int rows,
                                  int max_rows) {
  return bytes_or_zero([&] {
    const Layout at = pool_of(reinterpret_cast<void*>(16), 1, kv_heads, head_dim).at;
    check_sizes(at, heads, nseq, max_blocks, rows);
    PGD_CHECK(max_rows >= 0, kErrArg, "max_rows must not be negative");
    return attn_ws_bytes(at, heads, nseq, max_blocks, rows, max_rows);
  });
}

int pgd_attn_kv8_dev(pgd_dev* dev, const void* pool, int n_pages, int kv_heads, int head_dim, int heads, const void* q,
                     int ldq, int type, int nseq, const int* row_start, const int* lens, const int* block_tables,
                     int max_blocks, int rows, int max_rows, void* out, int ldo, const void* gate, int ldg, void* ws,
                     size_t ws_bytes) {
  return guard([&] {
    PGD_CHECK(dev, kErrArg, "null device");
    const Pool p = pool_of(pool, n_pages, kv_heads, head_dim);
    const Rows r = rows_of(p, heads, q, ldq, type, nseq, row_start, lens, block_tables, max_blocks, rows);
    PGD_CHECK(max_rows >= 0, kErrArg, "max_rows must not be negative");
    if (rows == 0 || nseq == 0) return;
    const Out o = out_of(r, p.at, out, ldo, gate, ldg);
    check_ws(ws, ws_bytes, attn_ws_bytes(p.at, heads, nseq, max_blocks, rows, max_rows));
    DeviceScope scope(dev);
    attn(p, r, max_rows, o, ws, dev->stream);
  });
}

size_t pgd_kv8_sparse_ws_bytes(int heads, int kv_heads, int head_dim, int rows, int max_blocks, int top) {
  return bytes_or_zero([&] {
    const Layout at = pool_of(reinterpret_cast<void*>(16), 1, kv_heads, head_dim).at;
    check_sizes(at, heads, 0, max_blocks, rows);
    check_list(at, heads, rows, max_blocks, top);
    return sparse_ws(at, heads, rows, max_blocks, top);
  });
}

int pgd_kv8_select_dev(pgd_dev* dev, const void* pool, int n_pages, int kv_heads, int head_dim, int heads,
                       const void* q, int ldq, int type, int nseq, const int* row_start, const int* lens,
                       const int* block_tables, int max_blocks, int rows, int top, int sinks, int recent, int* sel,
                       int* count, void* ws, size_t ws_bytes) {
  return guard([&] {
    PGD_CHECK(dev, kErrArg, "null device");
    const Pool p = pool_of(pool, n_pages, kv_heads, head_dim);
    const Rows r = rows_of(p, heads, q, ldq, type, nseq, row_start, lens, block_tables, max_blocks, rows);
    check_list(p.at, heads, rows, max_blocks, top);
    PGD_CHECK(sinks >= 0 && recent >= 0 && (int64_t)sinks + recent <= top, kErrArg,
              "sinks and recent must not be negative, nor more than top together");
    if (rows == 0 || nseq == 0) return;
    PGD_CHECK(sel && count, kErrArg, "null selection");
    check_ws(ws, ws_bytes, select_ws_bytes(p.at, rows, max_blocks));
    DeviceScope scope(dev);
    select(p, r, top, sinks, recent, sel, count, ws, dev->stream);
  });
}

int pgd_attn_kv8_sparse_dev(pgd_dev* dev, const void* pool, int n_pages, int kv_heads, int head_dim, int heads,
                            const void* q, int ldq, int type, int nseq, const int* row_start, const int* lens,
                            const int* block_tables, int max_blocks, int rows, int top, const int* sel,
                            const int* count, void* out, int ldo, const void* gate, int ldg, void* ws,
                            size_t ws_bytes) {
  return guard([&] {
    PGD_CHECK(dev, kErrArg, "null device");
    const Pool p = pool_of(pool, n_pages, kv_heads, head_dim);
    const Rows r = rows_of(p, heads, q, ldq, type, nseq, row_start, lens, block_tables, max_blocks, rows);
    check_list(p.at, heads, rows, max_blocks, top);
    if (rows == 0 || nseq == 0) return;
    PGD_CHECK(sel && count, kErrArg, "null selection");
    const Out o = out_of(r, p.at, out, ldo, gate, ldg);
    check_ws(ws, ws_bytes, attn_sparse_ws_bytes(p.at, heads, rows, top));
    DeviceScope scope(dev);
    attn_sparse(p, r, top, sel, count, o, ws, dev->stream);
  });
}

}  // extern "C"
