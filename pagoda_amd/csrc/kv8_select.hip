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

// The pages of a row's context (0 for none).
__device__ inline int row_pages(const Rows& r, int row, int& seq) {
  const RowSeq rs = row_seq(r, row);
  seq = rs.seq;
  return seq < 0 ? 0 : min((rs.seen(row) - 1) / kPage + (rs.seen(row) > 0 ? 1 : 0), r.max_blocks);
}

// Smallest exponent with top <= 127 * 2^e; 127 is 1.984375 * 2^6.
__device__ inline int holds127(float top) {
  const uint32_t b = __builtin_bit_cast(uint32_t, top);
  const int e = (int)(b >> 23) - 127 - 6 + ((b & 0x7fffffu) > 0x7e0000u ? 1 : 0);
  return e > kExpMin ? e : kExpMin;
}

// Workgroup: 64 TILES pages of one (row, KV head), 16 TILES a wave. The first bounds are on their way before q is
// turned into operands. Latency at few pages (one f32 row, 2049 pages: 4.2 us); 24 bf16 rows on 3000 to 60000
// positions, 4 heads of 128: 11.3 to 13 us, 2.3 TB/s.
template <int HD, int T, int TILES>
__global__ __launch_bounds__(256) void score_kernel(Pool p, Rows r, float* scores) {
  constexpr int kSegs = HD / 64, kPages = 64 * TILES;
  constexpr int kUnits = 16 * HD / 8, kRounds = kUnits > 256 ? kUnits / 256 : 1;
  __shared__ __align__(16) int8_t q8[2][kSegs][64][16];  // operand order: lane l = 16 kq + query
  __shared__ float tops[4];
  const int kv_heads = p.at.kv_heads, group = r.heads / kv_heads;
  const int strips = (r.max_blocks + kPages - 1) / kPages, unit = blockIdx.x / strips;
  const int row = unit / kv_heads, head = unit % kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n16 = lane & 15, kq = lane >> 4;
  auto finite = [](float v) { return fabsf(v) <= 3.402823466e38f ? v : 0.0f; };
  const int64_t q_at = (int64_t)row * r.ldq + (int64_t)head * group * HD;
  auto load_q = [&](int q0, int i, float (&x)[8]) {
    const int u = tid + i * 256;
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = 0;
    if (u < kUnits && q0 + u / (HD / 8) < group) load8<T>(r.q, q_at + (int64_t)q0 * HD + u * 8, x);
  };
  float x[kRounds][8];
#pragma unroll
  for (int i = 0; i < kRounds; i++) load_q(0, i, x[i]);
  int seq;
  const int pages = row_pages(r, row, seq);
  const int page0 = (int)(blockIdx.x % strips) * kPages;
  if (page0 >= pages) return;

  const int* table = r.block_tables + (int64_t)seq * r.max_blocks;
  int id[TILES];
#pragma unroll
  for (int i = 0; i < TILES; i++) {
    const int page = page0 + (i * 4 + wave) * 16 + n16;
    id[i] = page < pages ? table[page] : -1;
  }
  const size_t page_bytes = p.at.page_bytes(), bounds_at = p.at.bounds_at() + (size_t)head * 2 * HD + kq * 16,
               meta_at = p.at.meta_at() + (size_t)head * 4;
  i4 bound[2][kSegs];
  uint32_t meta;
  auto load_bounds = [&](int i) {
    const uint8_t* b = p.base + (size_t)(id[i] >= 0 && id[i] < p.n_pages ? id[i] : 0) * page_bytes;
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int s = 0; s < kSegs; s++) bound[w][s] = *reinterpret_cast<const i4*>(b + bounds_at + w * HD + s * 64);
    meta = *reinterpret_cast<const uint32_t*>(b + meta_at);
  };
  load_bounds(0);

  float most = 0;
#pragma unroll
  for (int i = 0; i < kRounds; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(finite(x[i][j])));
  for (int q0 = 16; q0 < group; q0 += 16)
    for (int i = 0; i < kRounds; i++) {
      float more[8];
      load_q(q0, i, more);
#pragma unroll
      for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(finite(more[j])));
    }
  most = lanes_max<64>(most);
  if (lane == 0) tops[wave] = most;
  __syncthreads();
  const float down = pow2(-holds127(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]))));

  int best[TILES];
#pragma unroll
  for (int i = 0; i < TILES; i++) best[i] = INT32_MIN;
  float scale[TILES];  // (a page outside the pool: -1)
  for (int q0 = 0; q0 < group; q0 += 16) {
    if (q0 > 0) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kRounds; i++) load_q(q0, i, x[i]);
      load_bounds(0);
    }
#pragma unroll
    for (int i = 0; i < kRounds; i++) {
      const int u = tid + i * 256, q = u / (HD / 8), g8 = u % (HD / 8);
      if (u < kUnits) {
        const int l = (g8 >> 1 & 3) * 16 + q;
        uint32_t pos[2] = {0, 0}, neg[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int v = (int)rintf(finite(x[i][j]) * down);
          pos[j / 4] |= (uint32_t)(max(v, 0) & 255) << (8 * (j & 3));
          neg[j / 4] |= (uint32_t)(min(v, 0) & 255) << (8 * (j & 3));
        }
        *reinterpret_cast<u2*>(&q8[0][g8 >> 3][l][(g8 & 1) * 8]) = u2{pos[0], pos[1]};
        *reinterpret_cast<u2*>(&q8[1][g8 >> 3][l][(g8 & 1) * 8]) = u2{neg[0], neg[1]};
      }
    }
    __syncthreads();
    i4 qa[2][kSegs];
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int s = 0; s < kSegs; s++) qa[w][s] = *reinterpret_cast<const i4*>(q8[w][s][lane]);
#pragma unroll
    for (int i = 0; i < TILES; i++) {
      i4 acc{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 2; w++)
#pragma unroll
        for (int s = 0; s < kSegs; s++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[w][s], bound[w][s], acc, 0, 0, 0);
      scale[i] = id[i] >= 0 && id[i] < p.n_pages ? pow2(Meta::ek(meta)) : -1.0f;
      if (i + 1 < TILES) load_bounds(i + 1);
      // acc[j]: query q0 + 4 kq + j with this lane's page
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (q0 + 4 * kq + j < group) best[i] = max(best[i], acc[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < TILES; i++) {
    const int v = quads_max(best[i]);
    const int page = page0 + (i * 4 + wave) * 16 + n16;
    if (kq == 0 && page < pages)
      scores[((int64_t)row * kv_heads + head) * r.max_blocks + page] = scale[i] > 0 ? (float)v * scale[i] : -INFINITY;
  }
}

constexpr int kPick = 1024;

// A float's order as that of whole numbers, zeros of both signs alike.
__device__ inline uint32_t order_of(float s) {
  uint32_t b = __builtin_bit_cast(uint32_t, s == 0 ? 0.0f : s);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Workgroup per (row, KV head): the lowest key that is taken, then the pages in order. A round counts the keys of
// a range in 2048 equal bins from its top and goes on with the bin that holds the last key taken; a bin
// of at most kRank keys is settled by counting, per key, those before it. Scores lie close together, and
// the first range is that of the keys themselves, so one round mostly does. Bound by the latency of its steps: 7 us
// for 128 of 2049 pages, 7.7 for 64 of up to 3750.
constexpr int kBins = 2 * kPick, kBinBits = __builtin_ctz(kBins), kRank = kPick, kHeld = 8;

__global__ __launch_bounds__(kPick) void pick_kernel(Rows r, int kv_heads, int top, int sinks, int recent,
                                                     const float* scores, int* sel, int* count) {
  __shared__ uint32_t lds[kBins > 2 * kRank ? kBins : 2 * kRank];  // bins, then (key, page) of the last bin
  __shared__ uint32_t part[2][kPick / 64];
  __shared__ int counts[kHeld * kPick / 64];
  __shared__ uint32_t chosen[4];  // bin, keys still to take, keys of the bin; keys listed
  const int row = blockIdx.x / kv_heads, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // (scores of pages past the row's are whatever the workspace held, and not looked at)
  const float* s = scores + (int64_t)blockIdx.x * r.max_blocks;
  float early[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; j++) {
    const int i = sinks + j * kPick + tid;
    early[j] = i < r.max_blocks ? s[i] : 0.0f;
  }
  int seq;
  const int pages = row_pages(r, row, seq);
  if (seq < 0) return;
  int* to = sel + (int64_t)blockIdx.x * top;
  const int take = min(top, pages);
  if (tid == 0) count[blockIdx.x] = take;
  for (int i = take + tid; i < top; i += kPick) to[i] = -1;
  if (take == pages) {
    for (int i = tid; i < pages; i += kPick) to[i] = i;
    return;
  }
  // Pages that are taken anyway are none of the keys.
  const int from = min(sinks, pages), until = max(pages - recent, from), forced = pages - (until - from);
  uint32_t held[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; j++) {
    const int i = from + j * kPick + tid;
    held[j] = i < until ? order_of(early[j]) : 0;  // (from is sinks, or no page is left)
  }
  // f(key, page) for this thread's keys
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < kHeld; j++) {
      const int i = from + j * kPick + tid;
      if (i < until) f(held[j], i);
    }
    for (int i = from + kHeld * kPick + tid; i < until; i += kPick) f(order_of(s[i]), i);
  };
  for (int i = tid; i < kBins; i += kPick) lds[i] = 0;
  if (tid == 0) chosen[3] = 0;
  uint32_t low = ~0u, high = 0;
  each([&](uint32_t k, int) { low = min(low, k), high = max(high, k); });
  low = lanes_min<64>(low);
  high = lanes_max<64>(high);
  if (lane == 0) part[0][wave] = low, part[1][wave] = high;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kPick / 64; w++) low = min(low, part[0][w]), high = max(high, part[1][w]);

  int need = take - forced;  // still to take among the keys of [low, high]; those above are taken
  int listed = 0;            // keys of the last bin, in lds
  while (need > 0) {
    const uint32_t span = high - low;
    const int shift = max(0, 32 - kBinBits - (span ? __builtin_clz(span) : 32));  // span >> shift < kBins
    each([&](uint32_t k, int) {
      if (k >= low && k <= high) atomicAdd(&lds[(high - k) >> shift], 1u);
    });
    __syncthreads();
    // thread t holds the bins 2 t and 2 t + 1
    const uint32_t a = lds[2 * tid], b = lds[2 * tid + 1];
    uint32_t upto = (uint32_t)wave_scan((int)(a + b));
    if (lane == 63) part[0][wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; w++) upto += part[0][w];
    const uint32_t before = upto - a - b;
    if (before < (uint32_t)need && (uint32_t)need <= upto) {
      const bool first = (uint32_t)need <= before + a;
      chosen[0] = 2 * tid + (first ? 0 : 1);
      chosen[1] = need - (first ? before : before + a);
      chosen[2] = first ? a : b;
    }
    __syncthreads();
    const uint32_t bin = chosen[0];
    need = (int)chosen[1];
    const int many = (int)chosen[2];
    high -= bin << shift;
    low = high - low >= (1u << shift) ? high - ((1u << shift) - 1) : low;
    if (many <= kRank || low == high) {
      listed = many;
      break;
    }
    for (int i = tid; i < kBins; i += kPick) lds[i] = 0;
    __syncthreads();
  }
  // Which of the last bin's keys: by rank if they are few; else they are all equal and the lowest pages win.
  const bool ranked = need > 0 && listed <= kRank;
  if (ranked) {
    each([&](uint32_t k, int i) {
      if (k >= low && k <= high) {
        const uint32_t at = atomicAdd(&chosen[3], 1u);
        lds[2 * at] = k;
        lds[2 * at + 1] = (uint32_t)i;
      }
    });
    __syncthreads();
  }
  auto taken = [&](uint32_t k, int i) {  // 1: taken, 2: one of too many equal keys, by page
    if (need == 0 || k < low) return 0;
    if (k > high) return 1;
    if (!ranked) return 2;
    int rank = 0;
    for (int j = 0; j < listed; j++) rank += lds[2 * j] > k || (lds[2 * j] == k && lds[2 * j + 1] < (uint32_t)i);
    return rank < need ? 1 : 0;
  };
  for (int i = tid; i < from; i += kPick) to[i] = i;
  for (int i = tid; i < pages - until; i += kPick) to[take - (pages - until) + i] = until + i;
  if (ranked && until - from <= kHeld * kPick) {
    // all keys are held: one count of every 64 pages, in page order
    uint64_t mine[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; j++) {
      const int i = from + j * kPick + tid;
      mine[j] = __ballot(i < until && taken(held[j], i) == 1);
      if (lane == 0) counts[j * (kPick / 64) + wave] = __popcll(mine[j]);
    }
    __syncthreads();
    static_assert(kHeld * kPick / 64 == 128, "two counts a lane");
    const int a = counts[2 * lane], b = counts[2 * lane + 1], upto = wave_scan(a + b);
#pragma unroll
    for (int j = 0; j < kHeld; j++) {
      const int e = j * (kPick / 64) + wave;  // (the same for the whole wave)
      const int pair_end = __builtin_amdgcn_readlane(upto, e >> 1), second = __builtin_amdgcn_readlane(b, e >> 1),
                first = __builtin_amdgcn_readlane(a, e >> 1);
      const int before = pair_end - second - (e & 1 ? 0 : first);
      if (mine[j] >> lane & 1)
        to[from + before + __popcll(mine[j] & ((1ull << lane) - 1))] = from + j * kPick + tid;
    }
    return;
  }
  int at = from, equal = 0;
  for (int j = 0; from + j * kPick < until; j++) {
    const int i = from + j * kPick + tid;
    int how = 0;
    if (i < until) {
      uint32_t k = 0;
      if (j < kHeld) {
#pragma unroll
        for (int h = 0; h < kHeld; h++) k = j == h ? held[h] : k;
      } else {
        k = order_of(s[i]);
      }
      how = taken(k, i);
    }
    const uint64_t sure = __ballot(how == 1), tie = __ballot(how == 2);
    __syncthreads();
    if (lane == 0) part[0][wave] = __popcll(sure), part[1][wave] = __popcll(tie);
    __syncthreads();
    int g = at, e = equal;
    for (int w = 0; w < kPick / 64; w++) {
      if (w < wave) g += part[0][w], e += part[1][w];
      at += part[0][w];
      equal += part[1][w];
    }
    const uint64_t below = (1ull << lane) - 1;
    g += __popcll(sure & below);
    e += __popcll(tie & below);
    if (how == 1 || (how == 2 && e < need)) to[g + min(e, ranked ? 0 : need)] = i;
  }
}

template <int HD, int TILES>
void score_of(const Pool& p, const Rows& r, float* scores, hipStream_t s) {
  const unsigned grid = (unsigned)(r.rows * p.at.kv_heads) * ((r.max_blocks + 64 * TILES - 1) / (64 * TILES));
  if (r.type == F32) score_kernel<HD, F32, TILES><<<grid, 256, 0, s>>>(p, r, scores);
  else if (r.type == F16) score_kernel<HD, F16, TILES><<<grid, 256, 0, s>>>(p, r, scores);
  else score_kernel<HD, BF16, TILES><<<grid, 256, 0, s>>>(p, r, scores);
  PGD_HIP(hipGetLastError());
}

template <int HD>
void score_hd(const Pool& p, const Rows& r, float* scores, hipStream_t s) {
  // 64 pages a workgroup while that makes few of them, 128 past that.
  if ((int64_t)r.rows * p.at.kv_heads * r.max_blocks <= 64 * 2048) score_of<HD, 1>(p, r, scores, s);
  else score_of<HD, 2>(p, r, scores, s);
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
