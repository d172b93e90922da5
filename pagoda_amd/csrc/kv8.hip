// kv8.hip — writing, reading and addressing the 8-bit paged KV cache.
//
// A (page, KV head) holds its keys as e4m3 codes times 2^ek and its values as codes
// times 2^ev, e the smallest exponent that holds the largest magnitude written to it
// (e never falls while the page fills; a row at place 0 starts the page anew). A power
// of two keeps every step exact but the one rounding to a code: x 2^-e is exact, and so
// is moving codes to a larger exponent down to where they leave e4m3's normal range.
// A factor amax / 448 would use at most one more bit of range, which a floating
// format does not turn into accuracy.
#include <climits>

#include "kv8_dev.h"

namespace pgd {
namespace kv8 {

namespace {

__device__ inline bool slot_ok(int slot, int n_pages) { return slot >= 0 && (slot >> 4) < n_pages; }

// One workgroup per (row, KV head); the row that is first of its page in the call
// takes the page and the rows that follow it there, the others end at once.
// The page is made in LDS and written whole: 32 hd bytes, whatever part is new.
template <int HD, int T>
__global__ __launch_bounds__(256) void append_kernel(Pool p, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                                     const int* slots, int rows) {
  constexpr int kGroups = HD / 8;                       // threads over a row, 8 dims each
  constexpr int kStep = 256 / kGroups < kPage ? 256 / kGroups : kPage;  // rows a pass
  constexpr int kPasses = kPage / kStep;
  __shared__ __align__(16) uint8_t code[2][kPage * HD];
  __shared__ uint32_t bad;
  __shared__ float top[2][4];
  const int head = blockIdx.y, row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

  const int first = slots[row];
  if (!slot_ok(first, p.n_pages)) return;
  const int s0 = first & 15;
  if (row > 0 && s0 > 0 && slots[row - 1] == first - 1) return;
  int n = 1;
  {
    const int i = lane & 15;
    const bool next = i > 0 && s0 + i < kPage && row + i < rows && slots[row + i] == first + i;
    const uint32_t run = (uint32_t)__ballot(next) & 0xffffu;
    n = __builtin_ctz(~(run >> 1)) + 1;
  }
  uint8_t* page = p.base + (size_t)(first >> 4) * p.at.page_bytes();
  u4* const dst[2] = {reinterpret_cast<u4*>(page + (size_t)head * p.at.head_bytes()),
                      reinterpret_cast<u4*>(page + (size_t)head * p.at.head_bytes() + kPage * HD)};
  uint32_t* meta = reinterpret_cast<uint32_t*>(page + p.at.meta_at()) + head;

  // what the page holds already
  const uint32_t m0 = s0 ? *meta : Meta::pack(kExpMin, kExpMin, 0);
  u4 old[2] = {u4{0, 0, 0, 0}, u4{0, 0, 0, 0}};
  if (s0 && tid < HD) {
    old[0] = dst[0][tid];
    old[1] = dst[1][tid];
  }

  // the new rows, and which of them have a non-finite value
  const int g = tid % kGroups, r = tid / kGroups;
  float x[2][kPasses][8];
  if (tid == 0) bad = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPasses; i++) {
    const int j = r + i * kStep;
    if (j < n && r < kStep) {
      load8<T>(k, (row + j) * ldk + head * HD + g * 8, x[0][i]);
      load8<T>(v, (row + j) * ldv + head * HD + g * 8, x[1][i]);
      bool ok = true;
#pragma unroll
      for (int w = 0; w < 2; w++)
#pragma unroll
        for (int d = 0; d < 8; d++) ok &= fabsf(x[w][i][d]) <= 3.402823466e38f;
      if (!ok) atomicOr(&bad, 1u << (s0 + j));
    }
  }
  __syncthreads();
  const uint32_t nan_new = bad;
  float most[2] = {0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kPasses; i++) {
    const int j = r + i * kStep;
    if (j < n && r < kStep && !(nan_new >> (s0 + j) & 1)) {
#pragma unroll
      for (int w = 0; w < 2; w++)
#pragma unroll
        for (int d = 0; d < 8; d++) most[w] = fmaxf(most[w], fabsf(x[w][i][d]));
    }
  }
#pragma unroll
  for (int w = 0; w < 2; w++) {
    most[w] = wave_max(most[w]);
    if (lane == 0) top[w][wave] = most[w];
  }
  __syncthreads();
  int e[2];
#pragma unroll
  for (int w = 0; w < 2; w++) {
    const int need = holds(fmaxf(fmaxf(top[w][0], top[w][1]), fmaxf(top[w][2], top[w][3])));
    e[w] = max(need, w ? Meta::ev(m0) : Meta::ek(m0));
  }

  // old codes at the new exponents, nothing at the places from s0 on
  if (tid < HD) {
    const int place_k = tid & 15, place_v = tid >> 4 & 3;
    const float down[2] = {pow2(max(Meta::ek(m0) - e[0], kExpMin)), pow2(max(Meta::ev(m0) - e[1], kExpMin))};
    uint32_t keep_v = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) keep_v |= 4 * place_v + j < s0 ? 0xffu << (8 * j) : 0u;
#pragma unroll
    for (int w = 0; w < 2; w++) {
      const uint32_t keep = w ? keep_v : place_k < s0 ? ~0u : 0u;
      u4 c;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const f4 u = of_codes(old[w][j] & keep) * down[w];
        c[j] = to_codes(u[0], u[1], u[2], u[3]);
      }
      reinterpret_cast<u4*>(code[w])[tid] = c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPasses; i++) {
    const int j = r + i * kStep;
    if (j < n && r < kStep) {
      const bool zero = nan_new >> (s0 + j) & 1;
      uint32_t c[2][2];
#pragma unroll
      for (int w = 0; w < 2; w++) {
        const float up = pow2(-e[w]);
        float u[8];
#pragma unroll
        for (int d = 0; d < 8; d++) u[d] = zero ? 0.0f : x[w][i][d] * up;
        c[w][0] = to_codes(u[0], u[1], u[2], u[3]);
        c[w][1] = to_codes(u[4], u[5], u[6], u[7]);
      }
      *reinterpret_cast<u2*>(code[0] + k_at(s0 + j, g * 8)) = u2{c[0][0], c[0][1]};
#pragma unroll
      for (int d = 0; d < 8; d++) code[1][v_at(s0 + j, g * 8 + d)] = (uint8_t)(c[1][d / 4] >> (8 * (d & 3)));
    }
  }
  __syncthreads();

  if (tid < HD) {
#pragma unroll
    for (int w = 0; w < 2; w++) dst[w][tid] = reinterpret_cast<const u4*>(code[w])[tid];
    // A code's order is that of its sign and magnitude. Bounds are outward in steps of
    // 4: codes reach 448, so they fit a signed byte, and a score of them is a sum of
    // whole numbers.
    int hi = INT_MIN, lo = INT_MAX;
    for (int j = 0; j < s0 + n; j++) {
      const int c = code[0][k_at(j, tid)], key = c & 128 ? -(c & 127) : c;
      hi = max(hi, key);
      lo = min(lo, key);
    }
    auto quarter = [](int key) {
      return of_codes((uint32_t)(key < 0 ? -key | 128 : key))[0] * 0.25f;
    };
    int8_t* bound = reinterpret_cast<int8_t*>(page + p.at.bounds_at()) + (size_t)head * 2 * HD;
    bound[tid] = (int8_t)ceilf(quarter(hi));
    bound[HD + tid] = (int8_t)floorf(quarter(lo));
  }
  if (tid == 0) *meta = Meta::pack(e[0], e[1], (Meta::nan(m0) & ((1u << s0) - 1u)) | nan_new);
}

// Positions by slot to f32 rows. A thread takes 4 dims of a row: of K one dword, of V a byte of each of
// four 16-byte runs.
__global__ __launch_bounds__(256) void read_kernel(Pool p, const int* slots, int64_t n4, float* k, int64_t ldk,
                                                   float* v, int64_t ldv) {
  const int hd = p.at.hd, per_row = p.at.kv_heads * hd / 4;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / per_row;
    const int c = (int)(i - row * per_row) * 4, head = c / hd, d = c - head * hd, slot = slots[row];
    if (!slot_ok(slot, p.n_pages)) continue;
    const uint8_t* page = p.base + (size_t)(slot >> 4) * p.at.page_bytes();
    const uint32_t m = reinterpret_cast<const uint32_t*>(page + p.at.meta_at())[head];
    const uint8_t* kc = page + (size_t)head * p.at.head_bytes();
    const uint8_t* vc = kc + kPage * hd;
    const int place = slot & 15;
    f4 a = of_codes(*reinterpret_cast<const uint32_t*>(kc + k_at(place, d))) * pow2(Meta::ek(m));
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) w |= (uint32_t)vc[v_at(place, d + j)] << (8 * j);
    f4 b = of_codes(w) * pow2(Meta::ev(m));
    if (Meta::nan(m) >> place & 1) a = b = f4{NAN, NAN, NAN, NAN};
    *reinterpret_cast<f4*>(k + row * ldk + c) = a;
    *reinterpret_cast<f4*>(v + row * ldv + c) = b;
  }
}

// ---- block tables and slot maps -------------------------------------------------

enum Status { kFits = 0, kNoPages = 1, kNoTable = 2, kNoRows = 3, kBadInput = 4 };

constexpr int kScan = 1024;

// Inclusive sums of two values over the workgroup's kScan threads.
__device__ inline void block_scan2(long long& a, long long& b, long long (*part)[2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long x = __shfl_up(a, o), y = __shfl_up(b, o);
    if (lane >= o) a += x, b += y;
  }
  __syncthreads();  // (part of the strip before has been read)
  if (lane == 63) part[wave][0] = a, part[wave][1] = b;
  __syncthreads();
  for (int w = 0; w < wave; w++) a += part[w][0], b += part[w][1];
}

// The sequence, position and slot of one row, from the row starts and tables written before.
__device__ inline void place_row(const Tables& t, int r) {
  int seq = -1, pos = -1, slot = -1;
  if (r < t.row_start[t.nseq]) {
    int lo = 0, hi = t.nseq;  // row_start[lo] <= r < row_start[hi]
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (t.row_start[mid] <= r) lo = mid;
      else hi = mid;
    }
    if (t.status[lo] == kFits) {
      seq = lo;
      pos = t.new_lens[lo] - t.counts[lo] + (r - t.row_start[lo]);
      const int page = t.tables[(int64_t)lo * t.max_blocks + pos / t.block];
      if (page >= 0 && page <= (INT_MAX - t.block) / t.block) slot = page * t.block + pos % t.block;
    }
  }
  t.seq_of_row[r] = seq;
  t.pos_of_row[r] = pos;
  t.slots[r] = slot;
}

// One workgroup over the sequences, in strips of kScan: what each needs, running sums of rows and pages,
// the pages into the tables; with ROWS the rows too.
template <bool ROWS>
__global__ __launch_bounds__(kScan) void tables_kernel(Tables t) {
  __shared__ long long part[kScan / 64][2];
  __shared__ long long carry[2];
  __shared__ int granted;
  const int tid = threadIdx.x;
  const int taken = t.taken[0];
  const long long avail = taken >= 0 && taken <= t.n_free ? t.n_free - taken : 0;
  if (tid == 0) carry[0] = carry[1] = 0, granted = 0;
  __syncthreads();
  for (int base = 0; base < t.nseq; base += kScan) {
    const int i = base + tid;
    int len = 0, count = 0, status = kFits, have = 0;
    long long need = 0, rows = 0;
    if (i < t.nseq) {
      len = t.lens[i];
      count = t.counts[i];
      if (len < 0 || count < 0) status = kBadInput;
      else {
        rows = count;
        have = (int)(((long long)len + t.block - 1) / t.block);
        const long long want = ((long long)len + count + t.block - 1) / t.block;
        if (want > t.max_blocks || (long long)len + count > INT_MAX) status = kNoTable;
        else need = want - have;
      }
    }
    // (Rows are laid out and pages counted for refused sequences too: whatever comes behind rows or
    // pages that do not fit has either none of its own or does not fit itself.)
    long long row_end = rows, page_end = need;
    block_scan2(row_end, page_end, part);
    row_end += carry[0];
    page_end += carry[1];
    if (status == kFits && row_end > t.rows) status = kNoRows;
    if (status == kFits && need > 0 && page_end > avail) status = kNoPages;
    if (i < t.nseq) {
      const long long start = row_end - rows;
      t.row_start[i] = (int)(start < t.rows ? start : t.rows);
      if (i == t.nseq - 1) t.row_start[t.nseq] = (int)(row_end < t.rows ? row_end : t.rows);
      t.status[i] = status;
      t.new_lens[i] = status == kFits ? len + count : len;
      if (status == kFits && need > 0) {
        const int* from = t.free_pages + taken + (page_end - need);
        int* to = t.tables + (int64_t)i * t.max_blocks + have;
        for (int j = 0; j < (int)need; j++) to[j] = from[j];
        atomicMax(&granted, (int)page_end);
      }
    }
    __syncthreads();  // (carry has been read)
    if (tid == kScan - 1) carry[0] = row_end, carry[1] = page_end;
    __syncthreads();
  }
  if (tid == 0) {
    if (t.nseq == 0) t.row_start[0] = 0;
    t.new_taken[0] = taken + granted;
  }
  if constexpr (ROWS) {
    __syncthreads();
    for (int r = tid; r < t.rows; r += kScan) place_row(t, r);
  }
}

__global__ __launch_bounds__(256) void place_rows_kernel(Tables t) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r < t.rows) place_row(t, r);
}

template <int HD>
void append_hd(const Pool& p, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, const int* slots,
               int rows, hipStream_t s) {
  const dim3 grid(rows, p.at.kv_heads);
  if (type == F32) append_kernel<HD, F32><<<grid, 256, 0, s>>>(p, k, ldk, v, ldv, slots, rows);
  else if (type == F16) append_kernel<HD, F16><<<grid, 256, 0, s>>>(p, k, ldk, v, ldv, slots, rows);
  else append_kernel<HD, BF16><<<grid, 256, 0, s>>>(p, k, ldk, v, ldv, slots, rows);
  PGD_HIP(hipGetLastError());
}

}  // namespace

void append(const Pool& p, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, const int* slots, int rows,
            hipStream_t s) {
  if (p.at.hd == 64) append_hd<64>(p, k, ldk, v, ldv, type, slots, rows, s);
  else if (p.at.hd == 128) append_hd<128>(p, k, ldk, v, ldv, type, slots, rows, s);
  else append_hd<256>(p, k, ldk, v, ldv, type, slots, rows, s);
}

void read(const Pool& p, const int* slots, int rows, float* k, int64_t ldk, float* v, int64_t ldv, hipStream_t s) {
  const int64_t n4 = (int64_t)rows * p.at.kv_heads * p.at.hd / 4;
  const int64_t blocks = (n4 + 255) / 256;
  read_kernel<<<(int)(blocks < (1 << 20) ? blocks : 1 << 20), 256, 0, s>>>(p, slots, n4, k, ldk, v, ldv);
  PGD_HIP(hipGetLastError());
}

void tables(const Tables& t, hipStream_t s) {
  // One launch while a workgroup places the rows in few rounds, a second one over the rows past that.
  const bool one = t.rows <= 2 * kScan;
  if (one) tables_kernel<true><<<1, kScan, 0, s>>>(t);
  else tables_kernel<false><<<1, kScan, 0, s>>>(t);
  PGD_HIP(hipGetLastError());
  if (!one) {
    place_rows_kernel<<<(t.rows + 255) / 256, 256, 0, s>>>(t);
    PGD_HIP(hipGetLastError());
  }
}

}  // namespace kv8
}  // namespace pgd
