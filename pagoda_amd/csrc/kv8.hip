// kv8.hip — writing, reading and addressing the 8-bit paged KV cache.
//
// A (page, KV head) holds its keys as e4m3 codes times 2^ek and its values as codes
// times 2^ev, e the smallest exponent that holds the largest magnitude written to it
// (e never falls while the page fills; a row at place 0 starts the page anew). A power
// of two keeps every step exact but the one rounding to a code: x 2^-e is exact, and so
// is moving codes to a larger exponent down to where they leave e4m3's normal range.
// A factor amax / 448 would use at most one more bit of range, which a floating
// format does not turn into accuracy.
#include <algorithm>
#include <climits>

#include "kv8_dev.h"

namespace pgd {
namespace kv8 {

namespace {

__device__ inline bool slot_ok(int slot, int n_pages) { return slot >= 0 && (slot >> 4) < n_pages; }

// Orders a wave's LDS accesses (the compiler's, too: the hardware runs them in order).
__device__ inline void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A workgroup per (ROWS rows, KV head). A row that is first of its page in the call
// takes the page and the rows that follow it there (up to 15 past the workgroup's own), the others are
// passed over. The page is made in LDS and written whole: 32 hd bytes, whatever part is new.
// Few rows: 4 us, one page's chain of slots, loads, maxima, codes and bounds. 8400 prompt rows (bf16, 4 heads of 256:
// 34 MB in, 17 out) 20 us, 2.6 TB/s: all pages are in flight at once, so they load, compute and store together;
// the bounds and the values' single bytes are 1.3 us of it each. A wave a page is slower (its ~2500 instructions).
template <int HD, int T, int ROWS>
__global__ __launch_bounds__(256) void append_kernel(Pool p, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                                     const int* slots, int rows) {
  constexpr int kGroups = HD / 8;                       // threads over a row, 8 dims each
  constexpr int kStep = 256 / kGroups < kPage ? 256 / kGroups : kPage;  // rows a pass
  constexpr int kPasses = kPage / kStep;
  __shared__ __align__(16) uint8_t code[2][kPage * HD];
  __shared__ uint32_t bad;
  __shared__ float top[2][4];
  const int head = blockIdx.y, row0 = blockIdx.x * ROWS, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = tid % kGroups, r = tid / kGroups;
  // lane l: the slot of row0 - 1 + l, as far as the last page may reach
  const int at = row0 - 1 + lane, near = lane < ROWS + 16 && at >= 0 && at < rows ? slots[at] : -1;
#pragma unroll 1
  for (int own = 0; own < ROWS; own++) {
    const int row = row0 + own;
    const int first = __builtin_amdgcn_readlane(near, own + 1), before = __builtin_amdgcn_readlane(near, own);
    const int s0 = first & 15;
    if (!slot_ok(first, p.n_pages) || (s0 > 0 && before == first - 1)) continue;
    // bit l: lane l goes on with the run
    const int i = lane - own - 1;
    const uint64_t run = __ballot(i > 0 && s0 + i < kPage && near == first + i) >> (own + 1);
    const int n = __builtin_ctzll(~(run >> 1)) + 1;
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
    float x[2][kPasses][8];
    __syncthreads();  // (the page before is out of LDS)
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
      most[w] = lanes_max<64>(most[w]);
      if (lane == 0) top[w][wave] = most[w];
    }
    __syncthreads();
    int e[2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
      const int need = holds(fmaxf(fmaxf(top[w][0], top[w][1]), fmaxf(top[w][2], top[w][3])));
      e[w] = max(need, w ? Meta::ev(m0) : Meta::ek(m0));
    }

    // old codes at the new exponents, nothing at the places from s0 on (which the rows of a full page cover)
    const bool full = s0 == 0 && n == kPage;
    if (!full && tid < HD) {
      const int place_k = tid & 15, place_v = tid >> 4 & 3;
      const float down[2] = {pow2(max(Meta::ek(m0) - e[0], kExpMin)), pow2(max(Meta::ev(m0) - e[1], kExpMin))};
      uint32_t keep_v = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) keep_v |= 4 * place_v + j < s0 ? 0xffu << (8 * j) : 0u;
#pragma unroll
      for (int w = 0; w < 2; w++) {
        u4 c = old[w] & (w ? keep_v : place_k < s0 ? ~0u : 0u);
        if (s0 && e[w] != (w ? Meta::ev(m0) : Meta::ek(m0)))
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const f4 u = of_codes(c[j]) * down[w];
            c[j] = to_codes(u[0], u[1], u[2], u[3]);
          }
        reinterpret_cast<u4*>(code[w])[tid] = c;
      }
    }
    if (!full) __syncthreads();
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
}

// Positions by slot to f32 rows. A thread takes 4 dims of a row: of K one dword, of V a byte of each of
// four 16-byte runs. 2.6 us for one row (latency).
__global__ __launch_bounds__(256) void read_kernel(Pool p, const int* slots, int64_t n4, float* k, int64_t ldk,
                                                   float* v, int64_t ldv) {
  const int hd = p.at.hd, per_row = p.at.kv_heads * hd / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n4) return;
  const int64_t row = i / per_row;
  const int c = (int)(i - row * per_row) * 4, head = c / hd, d = c - head * hd, slot = slots[row];
  if (!slot_ok(slot, p.n_pages)) return;
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

// The same for many rows, whose slots mostly follow each other: a wave per (16 rows, KV head) takes its
// rows run by run of one page, the page's codes through LDS. 8400 rows of 4 heads of 256: 17 us, 86 MB
// at 5.1 TB/s, which bounds it.
template <int HD>
__global__ __launch_bounds__(256) void read_runs_kernel(Pool p, const int* slots, int rows, float* k, int64_t ldk,
                                                        float* v, int64_t ldv) {
  constexpr int kLanes = HD / 4, kAtOnce = 64 / kLanes, kRuns = HD / 64;
  __shared__ __align__(16) uint8_t lds[4][2 * kPage * HD];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint8_t* const code = lds[wave];
  const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
  const int row0 = __builtin_amdgcn_readfirstlane((int)(unit / p.at.kv_heads)) * 16;
  const int head = __builtin_amdgcn_readfirstlane((int)(unit % p.at.kv_heads));
  if (row0 >= rows) return;
  const int i16 = lane & 15;
  const int mine = row0 + i16 < rows ? slots[row0 + i16] : -1;
  const int previous = __shfl(mine, i16 > 0 ? i16 - 1 : 0);
  // bit i: row i does not go on with the run of the row before it
  const uint32_t starts = ((uint32_t)__ballot(i16 == 0 || mine != previous + 1 || (mine & 15) == 0) & 0xffffu) | 1u << 16;
  const int sub = lane / kLanes, d = lane % kLanes * 4;
  for (int at = 0; at < 16;) {
    const int n = __builtin_ctz(starts >> (at + 1)) + 1;
    const int slot = __builtin_amdgcn_readlane(mine, at);
    if (slot_ok(slot, p.n_pages)) {
      const uint8_t* page = p.base + (size_t)(slot >> 4) * p.at.page_bytes();
      const uint32_t m = reinterpret_cast<const uint32_t*>(page + p.at.meta_at())[head];
      const u4* codes = reinterpret_cast<const u4*>(page + (size_t)head * p.at.head_bytes());
      u4 c[2 * kRuns];
#pragma unroll
      for (int i = 0; i < 2 * kRuns; i++) c[i] = codes[i * 64 + lane];
      wave_lds_fence();
#pragma unroll
      for (int i = 0; i < 2 * kRuns; i++) reinterpret_cast<u4*>(code)[i * 64 + lane] = c[i];
      wave_lds_fence();
      const float ks = pow2(Meta::ek(m)), vs = pow2(Meta::ev(m));
      for (int j = sub; j < n; j += kAtOnce) {
        const int place = (slot & 15) + j;
        f4 a = of_codes(*reinterpret_cast<const uint32_t*>(code + k_at(place, d))) * ks;
        uint32_t w = 0;
#pragma unroll
        for (int b = 0; b < 4; b++) w |= (uint32_t)code[kPage * HD + v_at(place, d + b)] << (8 * b);
        f4 b = of_codes(w) * vs;
        if (Meta::nan(m) >> place & 1) a = b = f4{NAN, NAN, NAN, NAN};
        const int64_t row = row0 + at + j;
        *reinterpret_cast<f4*>(k + row * ldk + head * HD + d) = a;
        *reinterpret_cast<f4*>(v + row * ldv + head * HD + d) = b;
      }
    }
    at += n;
  }
}

// ---- block tables and slot maps -------------------------------------------------

enum Status { kFits = 0, kNoPages = 1, kNoTable = 2, kNoRows = 3, kBadInput = 4 };

// Orders LDS accesses of a workgroup, and nothing in global memory: stores go on meanwhile.
__device__ inline void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Inclusive sums over a workgroup of N threads of values in [0, 2^31), and the totals.
template <int N>
__device__ inline void block_scan2(long long (&v)[2], long long (&total)[2], long long (*part)[2]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // (64 halves of 16 bits fit an int)
  auto scan = [](long long x) {
    return ((long long)wave_scan((int)(x >> 16)) << 16) + wave_scan((int)(x & 0xffff));
  };
  v[0] = scan(v[0]);
  v[1] = scan(v[1]);
  if (lane == 63) part[wave][0] = v[0], part[wave][1] = v[1];
  lds_barrier();
  long long before[2] = {0, 0};
  total[0] = total[1] = 0;
#pragma unroll
  for (int w = 0; w < N / 64; w++)
#pragma unroll
    for (int i = 0; i < 2; i++) {
      total[i] += part[w][i];
      if (w < wave) before[i] += part[w][i];
    }
  v[0] += before[0];
  v[1] += before[1];
}

// Every workgroup goes over the sequences in strips of N: what each needs, running sums of rows and pages. The
// first one writes what belongs to sequences (with `maps` row starts and status, with `lens` new lengths and
// the pages taken); with `maps` all enter their share of the pages into the tables and place rows_per rows each. Nothing
// is read that the call writes: a row's new page comes from the free list. The same input arrays as outputs
// (lengths, taken) need one workgroup, or `lens` in a launch behind.
// Bound by the latency of a load, a scan, a search and a load: 4.5 us for one sequence, 7.8 for 512 of 46000 rows.
template <int N>
__global__ __launch_bounds__(N) void tables_kernel(Tables t, int rows_per, bool maps, bool lens) {
  __shared__ long long part[N / 64][2];
  // the strip's rows and pages before each sequence, pages that it has (-1: gets none), its length (-1: refused)
  __shared__ int starts[N + 1], fresh[N + 1], have_of[N], len_of[N];
  __shared__ int granted;
  const int tid = threadIdx.x;
  const bool first = blockIdx.x == 0;
  const int row0 = blockIdx.x * rows_per, row1 = min(row0 + rows_per, t.rows);
  const int taken = t.taken[0];
  const long long avail = taken >= 0 && taken <= t.n_free ? t.n_free - taken : 0;
  if (tid == 0) granted = 0;
  long long carry[2] = {0, 0};
  for (int base = 0; base < t.nseq; base += N) {
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
    long long end[2] = {rows, need}, total[2];
    block_scan2<N>(end, total, part);
    const long long row_end = carry[0] + end[0], page_end = carry[1] + end[1];
    if (status == kFits && row_end > t.rows) status = kNoRows;
    if (status == kFits && need > 0 && page_end > avail) status = kNoPages;
    const bool got = status == kFits && need > 0;
    auto clamp_rows = [&](long long x) { return (int)(x < t.rows ? x : t.rows); };
    auto clamp_pages = [&](long long x) { return (int)(x < avail ? x : avail); };
    starts[tid] = clamp_rows(row_end - rows);
    fresh[tid] = clamp_pages(page_end - need);
    have_of[tid] = got ? have : -1;
    len_of[tid] = status == kFits ? len : -1;
    if (tid == N - 1) starts[N] = clamp_rows(row_end), fresh[N] = clamp_pages(page_end);
    if (got) atomicMax(&granted, (int)page_end);
    if (first && i < t.nseq) {
      if (maps) {
        t.row_start[i] = starts[tid];
        t.status[i] = status;
      }
      if (lens) t.new_lens[i] = status == kFits ? len + count : len;
    }
    carry[0] += total[0];
    carry[1] += total[1];
    lds_barrier();
    // the last of a strip's sequences that begins at or before x
    auto owner = [](const int* begin, int x) {
      int lo = 0, hi = N;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (begin[mid] <= x) lo = mid;
        else hi = mid;
      }
      return lo;
    };
    if (maps) {
      for (int64_t pg = fresh[0] + (int64_t)blockIdx.x * N + tid; pg < fresh[N]; pg += (int64_t)gridDim.x * N) {
        const int s = owner(fresh, (int)pg);
        if (have_of[s] >= 0)
          t.tables[(int64_t)(base + s) * t.max_blocks + have_of[s] + (pg - fresh[s])] = t.free_pages[taken + pg];
      }
      for (int r = max(row0, starts[0]) + tid; r < min(row1, starts[N]); r += N) {
        const int s = owner(starts, r);
        int seq = -1, pos = -1, slot = -1;
        if (len_of[s] >= 0) {
          seq = base + s;
          pos = len_of[s] + (r - starts[s]);
          const int at = pos / t.block;
          const int page = have_of[s] >= 0 && at >= have_of[s] ? t.free_pages[taken + fresh[s] + (at - have_of[s])]
                                                               : t.tables[(int64_t)seq * t.max_blocks + at];
          if (page >= 0 && page <= (INT_MAX - t.block) / t.block) slot = page * t.block + pos % t.block;
        }
        t.seq_of_row[r] = seq;
        t.pos_of_row[r] = pos;
        t.slots[r] = slot;
      }
    }
    lds_barrier();  // (the strip's arrays have been read)
  }
  lds_barrier();
  const int used = (int)(carry[0] < t.rows ? carry[0] : t.rows);
  if (first && tid == 0) {
    if (maps) t.row_start[t.nseq] = used;
    if (lens) t.new_taken[0] = taken + granted;
  }
  if (maps)
    for (int r = max(row0, used) + tid; r < row1; r += N) t.seq_of_row[r] = t.pos_of_row[r] = t.slots[r] = -1;
}

template <int HD, int ROWS>
void append_rows(const Pool& p, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, const int* slots,
                 int rows, hipStream_t s) {
  const dim3 grid((rows + ROWS - 1) / ROWS, p.at.kv_heads);
  if (type == F32) append_kernel<HD, F32, ROWS><<<grid, 256, 0, s>>>(p, k, ldk, v, ldv, slots, rows);
  else if (type == F16) append_kernel<HD, F16, ROWS><<<grid, 256, 0, s>>>(p, k, ldk, v, ldv, slots, rows);
  else append_kernel<HD, BF16, ROWS><<<grid, 256, 0, s>>>(p, k, ldk, v, ldv, slots, rows);
  PGD_HIP(hipGetLastError());
}

template <int HD>
void append_hd(const Pool& p, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, const int* slots,
               int rows, hipStream_t s) {
  // 256 decode rows take 13.7 us with a workgroup a row (and head), 18.7 with one of four, which takes pages one
  // after the other; 500 decode rows 21.2 and 24.9; 512 rows of a prompt, where most workgroups of a row have no page
  // of their own, 16.7 and 11.9 (with the read-back of 3 us and more, head_dim 256, 4 KV heads). Four rows a
  // workgroup or eight: 2048 and 4000 rows of a prompt 23.5 and 19.1, 37.0 and 29.5; 2000 decode rows 79 both, 4000
  // 153 and 162; but 1000 decode rows 42 and 49.
  if (rows <= 256) append_rows<HD, 1>(p, k, ldk, v, ldv, type, slots, rows, s);
  else if (rows < 2048) append_rows<HD, 4>(p, k, ldk, v, ldv, type, slots, rows, s);
  else append_rows<HD, 8>(p, k, ldk, v, ldv, type, slots, rows, s);
}

}  // namespace

void append(const Pool& p, const void* k, int64_t ldk, const void* v, int64_t ldv, int type, const int* slots, int rows,
            hipStream_t s) {
  if (p.at.hd == 64) append_hd<64>(p, k, ldk, v, ldv, type, slots, rows, s);
  else if (p.at.hd == 128) append_hd<128>(p, k, ldk, v, ldv, type, slots, rows, s);
  else append_hd<256>(p, k, ldk, v, ldv, type, slots, rows, s);
}

void read(const Pool& p, const int* slots, int rows, float* k, int64_t ldk, float* v, int64_t ldv, hipStream_t s) {
  // Runs of 9 rows (64 pages): one by one 10 us with their write, run by run 17, of 200 pages and more the same; a
  // prompt's 1000 rows the same, 2048 rows 19.2 and 17.5, 4000 rows 29.5 and 24.5.
  if (rows >= 2048) {
    const unsigned grid = (unsigned)(((int64_t)(rows + 15) / 16 * p.at.kv_heads + 3) / 4);
    if (p.at.hd == 64) read_runs_kernel<64><<<grid, 256, 0, s>>>(p, slots, rows, k, ldk, v, ldv);
    else if (p.at.hd == 128) read_runs_kernel<128><<<grid, 256, 0, s>>>(p, slots, rows, k, ldk, v, ldv);
    else read_runs_kernel<256><<<grid, 256, 0, s>>>(p, slots, rows, k, ldk, v, ldv);
  } else {
    const int64_t n4 = (int64_t)rows * p.at.kv_heads * p.at.hd / 4;
    read_kernel<<<(unsigned)((n4 + 255) / 256), 256, 0, s>>>(p, slots, n4, k, ldk, v, ldv);
  }
  PGD_HIP(hipGetLastError());
}

void tables(const Tables& t, hipStream_t s) {
  const bool in_place = t.new_lens == t.lens || t.new_taken == t.taken;
  // 512 rows a workgroup: half its threads' worth, the rest enter pages meanwhile (46000 rows of 512 sequences 7.9
  // us, with 1024 rows a workgroup 8.2).
  constexpr int kRows = 512;
  const int groups = (t.rows + kRows - 1) / kRows;
  auto go = [&](int n, bool maps, bool lens) {
    // (4.5 us of the kernel for one sequence with 256 threads, 5.8 with 1024; more rows than threads take longer)
    if (t.nseq <= 256 && t.rows <= 256) tables_kernel<256><<<n, 256, 0, s>>>(t, kRows, maps, lens);
    else tables_kernel<1024><<<n, 1024, 0, s>>>(t, kRows, maps, lens);
    PGD_HIP(hipGetLastError());
  };
  if (in_place && groups > 1) {
    go(groups, true, false);
    go(1, false, true);
  } else {
    go(std::max(groups, 1), true, true);
  }
}

}  // namespace kv8
}  // namespace pgd
