// kv8_select.hip — the pages that a row's heads attend: a cheap bound on q.k per page.
//
// For a (row, KV head): q8 = rint(q 2^-eq), eq the smallest exponent with all group
// heads' |q| <= 127 2^eq. For a page with key bounds hi, lo (codes in steps of 4) and
// exponent ek
//   score = 2^ek max over the group's heads of sum_d max(q8_d hi_d, q8_d lo_d),
// no key of the page has a larger q8.k. The sum is one product of [max(q8, 0) | min(q8, 0)]
// with [hi | lo] in whole numbers: below 256 * 127 * 112 < 2^24, so the score is exact in f32
// and the choice does not hang on the order of any sum. The `top` highest scores are
// taken, ties to the lower page; the first `sinks` and the last `recent` pages of
// the row's context always are.
#include "kv8_dev.h"

namespace pgd {
namespace kv8 {

namespace {

constexpr int kScorePages = 256;  // pages of a scoring workgroup, 64 a wave

// The sequence that owns a row and the pages of the row's context (0 for none).
__device__ inline int row_pages(const Rows& r, int row, int& seq) {
  const int lane = threadIdx.x & 63;
  seq = -1;
  for (int base = 0; base < r.nseq; base += 64) {
    const int i = base + lane;
    const uint64_t hit = __ballot(i < r.nseq && r.row_start[i] <= row && row < r.row_start[i + 1]);
    if (hit) {
      seq = base + __builtin_ctzll(hit);
      break;
    }
  }
  if (seq < 0) return 0;
  const long long seen = (long long)r.lens[seq] - ((long long)r.row_start[seq + 1] - 1 - row);
  if (seen <= 0) return 0;
  const long long pages = (seen + kPage - 1) / kPage;
  return (int)(pages < r.max_blocks ? pages : r.max_blocks);
}

// Smallest exponent with top <= 127 * 2^e; 127 is 1.984375 * 2^6.
__device__ inline int holds127(float top) {
  const uint32_t b = __builtin_bit_cast(uint32_t, top);
  const int e = (int)(b >> 23) - 127 - 6 + ((b & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return e > kExpMin ? e : kExpMin;
}

// Workgroup: kScorePages pages of one (row, KV head).
template <int HD, int T>
__global__ __launch_bounds__(256) void score_kernel(Pool p, Rows r, float* scores) {
  constexpr int kSegs = HD / 64;
  __shared__ __align__(16) int8_t q8[2][kSegs][64][16];  // operand order: lane l = 16 kq + query
  __shared__ float tops[4];
  const int kv_heads = p.at.kv_heads, group = r.heads / kv_heads;
  const int strips = (r.max_blocks + kScorePages - 1) / kScorePages, unit = blockIdx.x / strips;
  const int row = unit / kv_heads, head = unit % kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n16 = lane & 15, kq = lane >> 4;
  int seq;
  const int pages = row_pages(r, row, seq);
  const int page0 = (int)(blockIdx.x % strips) * kScorePages;
  if (page0 >= pages) return;

  auto finite = [](float v) { return fabsf(v) <= 3.402823466e38f ? v : 0.0f; };
  const int64_t q_at = (int64_t)row * r.ldq + (int64_t)head * group * HD;
  float most = 0;
  for (int i = tid; i < group * HD / 8; i += 256) {
    float x[8];
    load8<T>(r.q, q_at + i * 8, x);
#pragma unroll
    for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(finite(x[j])));
  }
  most = wave_max(most);
  if (lane == 0) tops[wave] = most;
  __syncthreads();
  const float down = pow2(-holds127(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]))));

  int best[kScorePages / 64];
#pragma unroll
  for (int i = 0; i < kScorePages / 64; i++) best[i] = INT32_MIN;
  const int* table = r.block_tables + (int64_t)seq * r.max_blocks;
  for (int q0 = 0; q0 < group; q0 += 16) {
    __syncthreads();
    for (int u = tid; u < 16 * HD / 8; u += 256) {
      const int q = u / (HD / 8), g8 = u % (HD / 8);
      float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (q0 + q < group) load8<T>(r.q, q_at + (int64_t)(q0 + q) * HD + g8 * 8, x);
      const int l = (g8 >> 1 & 3) * 16 + q;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int v = (int)rintf(finite(x[j]) * down);
        q8[0][g8 >> 3][l][(g8 & 1) * 8 + j] = (int8_t)max(v, 0);
        q8[1][g8 >> 3][l][(g8 & 1) * 8 + j] = (int8_t)min(v, 0);
      }
    }
    __syncthreads();
    i4 qa[2][kSegs];
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int s = 0; s < kSegs; s++) qa[w][s] = *reinterpret_cast<const i4*>(q8[w][s][lane]);
#pragma unroll
    for (int i = 0; i < kScorePages / 64; i++) {
      const int page = page0 + wave * 64 + i * 16 + n16;
      const int id = page < pages ? table[page] : -1;
      const bool ok = id >= 0 && id < p.n_pages;
      const int8_t* b = reinterpret_cast<const int8_t*>(p.base + (size_t)(ok ? id : 0) * p.at.page_bytes() +
                                                         p.at.bounds_at()) + (size_t)head * 2 * HD;
      i4 acc{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 2; w++)
#pragma unroll
        for (int s = 0; s < kSegs; s++) {
          const i4 bound = *reinterpret_cast<const i4*>(b + w * HD + s * 64 + kq * 16);
          acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[w][s], bound, acc, 0, 0, 0);
        }
      // acc[j]: query q0 + 4 kq + j with this lane's page
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (q0 + 4 * kq + j < group) best[i] = max(best[i], acc[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < kScorePages / 64; i++) {
    int v = best[i];
    v = max(v, __shfl_xor(v, 16));
    v = max(v, __shfl_xor(v, 32));
    const int page = page0 + wave * 64 + i * 16 + n16;
    if (kq == 0 && page < pages) {
      const int id = table[page];
      float score = -INFINITY;  // (a page outside the pool)
      if (id >= 0 && id < p.n_pages) {
        const uint32_t m = reinterpret_cast<const uint32_t*>(p.base + (size_t)id * p.at.page_bytes() + p.at.meta_at())[head];
        score = (float)v * pow2(Meta::ek(m));
      }
      scores[((int64_t)row * kv_heads + head) * r.max_blocks + page] = score;
    }
  }
}

constexpr int kPick = 1024;

// A float's order as that of whole numbers, zeros of both signs alike.
__device__ inline uint32_t order_of(float s) {
  uint32_t b = __builtin_bit_cast(uint32_t, s == 0 ? 0.0f : s);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Workgroup per (row, KV head): the threshold by four rounds over the keys' bytes, highest first, then
// the pages above it, and the lowest ones that equal it, in page order.
__global__ __launch_bounds__(kPick) void pick_kernel(Rows r, int kv_heads, int top, int sinks, int recent,
                                                     const float* scores, int* sel, int* count) {
  __shared__ int bins[256];
  __shared__ int chosen, rest;
  __shared__ int wave_gt[kPick / 64], wave_eq[kPick / 64];
  const int row = blockIdx.x / kv_heads, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int seq;
  const int pages = row_pages(r, row, seq);
  if (seq < 0) return;
  const float* s = scores + (int64_t)blockIdx.x * r.max_blocks;
  int* to = sel + (int64_t)blockIdx.x * top;
  const int take = min(top, pages);
  if (tid == 0) count[blockIdx.x] = take;
  for (int i = take + tid; i < top; i += kPick) to[i] = -1;
  if (take == pages) {
    for (int i = tid; i < pages; i += kPick) to[i] = i;
    return;
  }
  auto key = [&](int i) { return i < sinks || i >= pages - recent ? ~0u : order_of(s[i]); };
  uint32_t prefix = 0;
  int need = take;  // still to take among the keys that begin with prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) bins[tid] = 0;
    __syncthreads();
    for (int i = tid; i < pages; i += kPick) {
      const uint32_t k = key(i);
      if (shift == 24 || k >> (shift + 8) == prefix) atomicAdd(&bins[k >> shift & 255], 1);
    }
    __syncthreads();
    if (wave == 0) {
      // lane l holds the bins 255 - 4 l .. 252 - 4 l, highest first
      int v[4], sum = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) sum += v[j] = bins[255 - 4 * lane - j];
      int upto = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(upto, o);
        if (lane >= o) upto += x;
      }
      int before = upto - sum;
      if (before < need && need <= upto) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (before < need && need <= before + v[j]) chosen = 255 - 4 * lane - j, rest = need - before;
          before += v[j];
        }
      }
    }
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)chosen;
    need = rest;
  }
  int at = 0, equal = 0;
  for (int base = 0; base < pages; base += kPick) {
    const int i = base + tid;
    const uint32_t k = i < pages ? key(i) : 0;
    const uint64_t gt = __ballot(i < pages && k > prefix), eq = __ballot(i < pages && k == prefix);
    if (lane == 0) wave_gt[wave] = __popcll(gt), wave_eq[wave] = __popcll(eq);
    __syncthreads();
    int g = at, e = equal;
    for (int w = 0; w < wave; w++) g += wave_gt[w], e += wave_eq[w];
    const uint64_t below = (1ull << lane) - 1;
    const int my_gt = g + __popcll(gt & below), my_eq = e + __popcll(eq & below);
    const int place = my_gt + min(my_eq, need);
    if ((gt >> lane & 1) || ((eq >> lane & 1) && my_eq < need)) to[place] = i;
    for (int w = 0; w < kPick / 64; w++) at += wave_gt[w], equal += wave_eq[w];
    __syncthreads();
  }
}

template <int HD>
void score_hd(const Pool& p, const Rows& r, float* scores, hipStream_t s) {
  const unsigned grid = (unsigned)(r.rows * p.at.kv_heads) * ((r.max_blocks + kScorePages - 1) / kScorePages);
  if (r.type == F32) score_kernel<HD, F32><<<grid, 256, 0, s>>>(p, r, scores);
  else if (r.type == F16) score_kernel<HD, F16><<<grid, 256, 0, s>>>(p, r, scores);
  else score_kernel<HD, BF16><<<grid, 256, 0, s>>>(p, r, scores);
  PGD_HIP(hipGetLastError());
}

}  // namespace

size_t select_ws_bytes(const Layout& at, int rows, int max_blocks) {
  return (size_t)rows * at.kv_heads * max_blocks * sizeof(float);
}

void select(const Pool& p, const Rows& r, int top, int sinks, int recent, int* sel, int* count, void* ws, hipStream_t s) {
  float* scores = static_cast<float*>(ws);
  if (p.at.hd == 64) score_hd<64>(p, r, scores, s);
  else if (p.at.hd == 128) score_hd<128>(p, r, scores, s);
  else score_hd<256>(p, r, scores, s);
  pick_kernel<<<r.rows * p.at.kv_heads, kPick, 0, s>>>(r, p.at.kv_heads, top, sinks, recent, scores, sel, count);
  PGD_HIP(hipGetLastError());
}

}  // namespace kv8
}  // namespace pgd
