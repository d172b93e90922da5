// attn_kv8.hip — causal GQA attention over the 8-bit paged KV cache: all pages of a
// sequence, or per (row, KV head) the pages of a list.
//
// For a query q of a row at position p:  o = sum_j w_j v_j / sum_j w_j over j <= p,
// w_j = exp(q.k_j / sqrt(hd)), with k_j = 2^ek codes, v_j = 2^ev codes per page and head.
// Per two pages (32 positions) and a tile of 16 queries (rows x group heads):
//   S[pos][query]  = K codes . q        16x16x32 bf16 products over hd / 32 steps
//   t = S 2^ek log2(e) / sqrt(hd), running maximum m and sum l in f32
//   O[dim][query] += V codes^T . (2^(t - m) 2^ev)   the same products over the 32 positions
// Codes convert to bf16 exactly. q enters exactly as bf16 terms (f32 three, f16 two,
// bf16 itself); the weights enter as three (f32) or two: each term leaves at most 2^-8 of what it
// is given, so f32 rows lose nothing that f32 sums keep, and the weights of f16 and bf16
// rows are held to 2^-16, well below what their results round to (one term would add as much
// error to bf16 results as their own rounding).
// The lane that holds a score holds it as the operand of the second product: lane
// (query n = l % 16, kq = l / 16) has positions 4 kq .. 4 kq + 3 of both pages, which
// are the 8 that a lane of the second product's operand takes, and its results are
// columns n too, so m, l and the rescaling stay in the lane but for one maximum
// over the four kq.
//
// Split: work is one list of (sequence, chunk of pages, KV head, tile) that every
// workgroup derives for itself from the row starts and lengths on the device, so a call
// needs no plan from the host. The chunk length makes about kItems items of all.
// In an item the four waves take pairs of pages in turn, each with its own m, l and O,
// joined in LDS. Items of a context of one chunk write results, the others partial sums that the merge kernel
// adds in chunk order.
#include <climits>

#include "kv8_dev.h"

namespace pgd {
namespace kv8 {

namespace {

constexpr int kItems = 1024;   // items that contexts are cut into, about
constexpr int kMinChunk = 16;  // pages: fewer would be more joining than reading

template <int T>
constexpr int kTerms = T == F32 ? 3 : T == F16 ? 2 : 1;  // of a query
template <int T>
constexpr int kWeightTerms = T == F32 ? 3 : 2;

// x as T terms of 8 bits, each the truncation of what is left (exact for what T is chosen for).
template <int T>
__device__ inline void split_trunc(const float (&x)[8], b8 (&out)[kTerms<T>]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; j++) r[j] = x[j];
#pragma unroll
  for (int k = 0; k < kTerms<T>; k++) {
    u4 w;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const uint32_t a = __builtin_bit_cast(uint32_t, r[j]), b = __builtin_bit_cast(uint32_t, r[j + 1]);
      w[j / 2] = (a >> 16) | (b & 0xffff0000u);
      r[j] -= __builtin_bit_cast(float, a & 0xffff0000u);
      r[j + 1] -= __builtin_bit_cast(float, b & 0xffff0000u);
    }
    out[k] = __builtin_bit_cast(b8, w);
  }
}

// x as terms rounded to nearest.
template <int T>
__device__ inline void split_near(const float (&x)[8], b8 (&out)[kWeightTerms<T>]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; j++) r[j] = x[j];
#pragma unroll
  for (int k = 0; k < kWeightTerms<T>; k++) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      out[k][j] = (__bf16)r[j];
      if (k + 1 < kWeightTerms<T>) r[j] -= (float)out[k][j];
    }
  }
}

// Eight codes as bf16.
__device__ inline b8 of_codes8(uint32_t lo, uint32_t hi) {
  const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const b2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const b2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return b8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ---- the list of items ------------------------------------------------------------

struct Seq {
  int row0, n;      // its rows
  int len;          // positions as given
  int ctx, pages;   // positions that the table holds, and their pages
  int tiles;        // query tiles of a KV head
};

__device__ inline Seq seq_at(const Rows& r, int group, int tile_queries, int i) {
  Seq s;
  const int a = min(max(r.row_start[i], 0), r.rows), b = min(max(r.row_start[i + 1], 0), r.rows);
  s.row0 = a;
  s.n = max(b - a, 0);
  s.len = r.lens[i];
  const long long most = (long long)r.max_blocks * kPage;
  s.ctx = (int)min((long long)max(s.len, 0), most);
  s.pages = (int)(((long long)s.ctx + kPage - 1) / kPage);
  s.tiles = (int)(((long long)s.n * group + tile_queries - 1) / tile_queries);
  return s;
}

__device__ inline int chunks_of(int pages, int chunk) { return pages > 0 ? (pages + chunk - 1) / chunk : 1; }

__device__ inline long long wave_sum64(long long v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ inline long long wave_scan64(long long v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long x = __shfl_up(v, o);
    if (lane >= o) v += x;
  }
  return v;
}

// Pages of a chunk: a multiple of 8 (a pair for each of four waves) that cuts all tiles' pages into at most kItems
// full chunks.
__device__ inline int chunk_of(long long tile_pages) {
  const long long c = (tile_pages + kItems - 1) / kItems;
  return (int)min(max((c + 7) & ~7ll, (long long)kMinChunk), (long long)INT_MAX / 2);
}

struct Found {
  Seq s;
  int seq;
  int chunk;       // pages of a chunk
  int item, slot;  // the sequence's first item, and its first partial sum if it has several chunks
};

// The sequence of an item (BY_ROW: of a row), as every wave works it out for itself, 64 sequences
// at a time. Returns false past the last.
template <bool BY_ROW>
__device__ inline bool find(const Rows& r, int kv_heads, int group, int tile_queries, int key, Found& f) {
  const int lane = threadIdx.x & 63;
  long long all = 0;
  for (int base = 0; base < r.nseq; base += 64) {
    const int i = base + lane;
    if (i < r.nseq) {
      const Seq s = seq_at(r, group, tile_queries, i);
      all += (long long)s.tiles * s.pages;
    }
  }
  f.chunk = chunk_of(wave_sum64(all) * kv_heads);
  long long before = 0;  // items in the low half, partial sums in the high one
  for (int base = 0; base < r.nseq; base += 64) {
    const int i = base + lane;
    Seq s{};
    long long mine = 0;
    if (i < r.nseq) {
      s = seq_at(r, group, tile_queries, i);
      const int chunks = chunks_of(s.pages, f.chunk);
      const long long items = (long long)s.tiles * chunks * kv_heads;
      mine = items | (chunks > 1 ? items << 32 : 0);
    }
    const long long upto = wave_scan64(mine) + before;
    const long long from = upto - mine;
    const int lo = (int)(uint32_t)from, hi = (int)(uint32_t)upto;
    const bool here = BY_ROW ? key >= s.row0 && key < s.row0 + s.n : key >= lo && key < hi;
    const uint64_t hit = __ballot(here);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      f.s.row0 = __builtin_amdgcn_readlane(s.row0, src);
      f.s.n = __builtin_amdgcn_readlane(s.n, src);
      f.s.len = __builtin_amdgcn_readlane(s.len, src);
      f.s.ctx = __builtin_amdgcn_readlane(s.ctx, src);
      f.s.pages = __builtin_amdgcn_readlane(s.pages, src);
      f.s.tiles = __builtin_amdgcn_readlane(s.tiles, src);
      f.item = __builtin_amdgcn_readlane(lo, src);
      f.slot = __builtin_amdgcn_readlane((int)(from >> 32), src);
      f.seq = base + src;
      return true;
    }
    before = ((long long)__builtin_amdgcn_readlane((int)(upto >> 32), 63) << 32) |
             (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)upto, 63);
  }
  return false;
}

// The sequence that owns a row: its index, -1 without one.
__device__ inline int seq_of(const Rows& r, int row) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < r.nseq; base += 64) {
    const int i = base + lane;
    const uint64_t hit = __ballot(i < r.nseq && r.row_start[i] <= row && row < r.row_start[i + 1]);
    if (hit) return base + __builtin_ctzll(hit);
  }
  return -1;
}

// ---- results ------------------------------------------------------------------------

template <int T>
__device__ inline f4 load4(const void* p, int64_t i) {
  if constexpr (T == F32) return *reinterpret_cast<const f4*>(static_cast<const float*>(p) + i);
  const u2 w = *reinterpret_cast<const u2*>(static_cast<const uint16_t*>(p) + i);
  f4 x;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const uint32_t h = j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu;
    x[j] = T == F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)h) : __builtin_bit_cast(float, h << 16);
  }
  return x;
}

// Four dims of a query's result: gate, rounding, store.
template <int T>
__device__ inline void store4(const Out& o, int64_t row, int64_t col, f4 x) {
  if (o.gate) {
    const f4 g = load4<T>(o.gate, row * o.ldg + col);
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = x[j] / (1.0f + __builtin_amdgcn_exp2f(g[j] * -1.44269504088896f));
  }
  if constexpr (T == F32) {
    *reinterpret_cast<f4*>(static_cast<float*>(o.out) + row * o.ldo + col) = x;
  } else {
    u2 w;
#pragma unroll
    for (int j = 0; j < 4; j += 2) {
      uint32_t a, b;
      if constexpr (T == F16) {
        a = __builtin_bit_cast(uint16_t, (_Float16)x[j]);
        b = __builtin_bit_cast(uint16_t, (_Float16)x[j + 1]);
      } else {
        a = __builtin_bit_cast(uint16_t, (__bf16)x[j]);
        b = __builtin_bit_cast(uint16_t, (__bf16)x[j + 1]);
      }
      w[j / 2] = a | b << 16;
    }
    *reinterpret_cast<u2*>(static_cast<uint16_t*>(o.out) + row * o.ldo + col) = w;
  }
}

// Partial sums: per slot and query O[hd], and behind all slots' O the pairs (m, l).
struct Partials {
  float* o;
  f2* ml;
};
template <int HD>
__device__ __host__ inline Partials partials_at(void* ws, int slots, int queries) {
  float* o = static_cast<float*>(ws);
  return Partials{o, reinterpret_cast<f2*>(o + (size_t)slots * queries * HD)};
}

struct List {
  const int *sel, *count;
  int top, chunk, chunks;  // pages of a chunk and chunks of a full list
};

// ---- the item kernel ----------------------------------------------------------------

template <int HD, int T, int NT, bool LIST>
__global__ __launch_bounds__(256) void item_kernel(Pool p, Rows r, Out out, List list, void* ws, int slots) {
  constexpr int kSegs = HD / 64, kSteps = HD / 32, kTiles = HD / 16, kQueries = 16 * NT, kN = kTerms<T>,
                kW = kWeightTerms<T>;
  constexpr int kQBytes = NT * kN * kSteps * 1024, kJoinBytes = 4 * kTiles * 1024;
  __shared__ __align__(16) uint8_t lds[kQBytes > kJoinBytes ? kQBytes : kJoinBytes];
  __shared__ f2 lds_ml[4][kQueries];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, kq = lane >> 4;
  const int kv_heads = p.at.kv_heads, group = r.heads / kv_heads;

  // which pages, head and queries
  int seq_table = 0, head, tile, page0, page1, row0, nrows, len, ctx, slot;
  const int* pages_list = nullptr;
  if constexpr (LIST) {
    const int tiles = (group + 15) / 16;
    int b = blockIdx.x;
    const int c = b % list.chunks;
    b /= list.chunks;
    tile = b % tiles;
    b /= tiles;
    head = b % kv_heads;
    const int row = b / kv_heads;
    const int seq = seq_of(r, row);
    if (seq < 0) return;
    const int count = min(max(list.count[(int64_t)row * kv_heads + head], 0), list.top);
    const int have = chunks_of(count, list.chunk);
    if (c >= have) return;
    page0 = c * list.chunk;
    page1 = min(page0 + list.chunk, count);
    pages_list = list.sel + ((int64_t)row * kv_heads + head) * list.top;
    seq_table = seq;
    row0 = row;
    nrows = 1;
    // (as the last of the rows up to this one)
    len = r.lens[seq] - (r.row_start[seq + 1] - 1 - row);
    ctx = (int)min((long long)max(len, 0), (long long)r.max_blocks * kPage);
    slot = have > 1 ? blockIdx.x : -1;
  } else {
    Found f;
    if (!find<false>(r, kv_heads, group, kQueries, blockIdx.x, f)) return;
    int local = blockIdx.x - f.item;
    const int chunks = chunks_of(f.s.pages, f.chunk);
    slot = chunks > 1 ? f.slot + local : -1;
    if (slot >= slots) return;  // (rows that belong to several sequences)
    tile = local % f.s.tiles;
    local /= f.s.tiles;
    head = local % kv_heads;
    const int c = local / kv_heads;
    page0 = c * f.chunk;
    page1 = min(page0 + f.chunk, f.s.pages);
    row0 = f.s.row0;
    nrows = f.s.n;
    len = f.s.len;
    ctx = f.s.ctx;
    seq_table = f.seq;
  }
  const int* table = r.block_tables + (int64_t)seq_table * r.max_blocks;

  // the tile's queries as operands: per (query tile, term, step) lane l's 16 bytes at 16 l
  for (int u = tid; u < kQueries * HD / 8; u += 256) {
    const int g8 = u % (HD / 8), q = u / (HD / 8);  // 8 dims of one query
    const int qi = tile * kQueries + q;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (qi < nrows * group) load8<T>(r.q, (int64_t)(row0 + qi / group) * r.ldq + (head * group + qi % group) * HD + g8 * 8, x);
    b8 t[kN];
    split_trunc<T>(x, t);
    // dims 64 seg + 16 kq + 8 half
    const int step = (g8 >> 3) * 2 + (g8 & 1), k4 = g8 >> 1 & 3;
#pragma unroll
    for (int k = 0; k < kN; k++)
      reinterpret_cast<b8*>(lds)[(((q >> 4) * kN + k) * kSteps + step) * 64 + k4 * 16 + (q & 15)] = t[k];
  }
  // positions that a lane's queries see
  int lim[NT];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    const int qi = tile * kQueries + t * 16 + n16;
    lim[t] = qi < nrows * group ? (int)min((long long)len - nrows + qi / group + 1, (long long)ctx) : 0;
  }
  __syncthreads();

  const float scale = 1.44269504088896340736f / sqrtf((float)HD);
  float m[NT], l[NT];
  f4 o[NT][kTiles];
#pragma unroll
  for (int t = 0; t < NT; t++) {
    m[t] = -INFINITY;
    l[t] = 0;
#pragma unroll
    for (int i = 0; i < kTiles; i++) o[t][i] = f4{0, 0, 0, 0};
  }

  // This wave's pairs are pages page0 + 2 (wave + 4 it) and the next; a lane holds one of its next 64 pages.
  const int pairs = (page1 - page0 - 2 * wave + 7) / 8;
  int my_index = 0, my_id = 0;
  auto refill = [&](int it) {
    const int i = page0 + 2 * (wave + 4 * (it + (lane >> 1))) + (lane & 1);
    my_index = -1;
    my_id = -1;
    if (i < page1) {
      my_index = LIST ? pages_list[i] : i;
      if (my_index >= 0 && my_index < r.max_blocks) {
        const int id = table[my_index];
        my_id = id >= 0 && id < p.n_pages ? id : -2;  // -2: attending it makes NaN
      } else {
        my_index = -1;
      }
    }
  };
  struct Page {
    int index, id;
    uint32_t meta;
    const uint8_t* at;
  };
  const size_t page_bytes = p.at.page_bytes(), head_at = (size_t)head * p.at.head_bytes(),
               meta_at = p.at.meta_at() + (size_t)head * 4;
  auto page_of = [&](int it, int which) {
    Page g;
    const int j = 2 * (it & 31) + which;
    g.index = __builtin_amdgcn_readlane(my_index, j);
    g.id = __builtin_amdgcn_readlane(my_id, j);
    const uint8_t* base = p.base + (size_t)max(g.id, 0) * page_bytes;
    g.at = base + head_at;
    g.meta = *reinterpret_cast<const uint32_t*>(base + meta_at);
    return g;
  };
  u4 kc[2][kSegs], vc[2][kSegs];
  auto load_k = [&](const Page (&g)[2]) {
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int s = 0; s < kSegs; s++) kc[w][s] = reinterpret_cast<const u4*>(g[w].at)[s * 64 + lane];
  };
  auto load_v = [&](const Page (&g)[2]) {
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int s = 0; s < kSegs; s++) vc[w][s] = reinterpret_cast<const u4*>(g[w].at + kPage * HD)[s * 64 + lane];
  };

  Page cur[2], next[2];
  if (pairs > 0) {
    refill(0);
    cur[0] = page_of(0, 0);
    cur[1] = page_of(0, 1);
    load_k(cur);
    load_v(cur);
  }
  for (int it = 0; it < pairs; it++) {
    const bool more = it + 1 < pairs;
    if (more) {
      if (((it + 1) & 31) == 0) refill(it + 1);
      next[0] = page_of(it + 1, 0);
      next[1] = page_of(it + 1, 1);
    }
    f4 sc[NT][2];
    {
      f4 acc[NT][2][kN];
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
          for (int k = 0; k < kN; k++) acc[t][w][k] = f4{0, 0, 0, 0};
#pragma unroll
      for (int step = 0; step < kSteps; step++) {
        const int s = step >> 1, h = step & 1;
        const b8 a0 = of_codes8(kc[0][s][2 * h], kc[0][s][2 * h + 1]);
        const b8 a1 = of_codes8(kc[1][s][2 * h], kc[1][s][2 * h + 1]);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int k = 0; k < kN; k++) {
            const b8 q = reinterpret_cast<const b8*>(lds)[((t * kN + k) * kSteps + step) * 64 + lane];
            acc[t][0][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a0, q, acc[t][0][k], 0, 0, 0);
            acc[t][1][k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a1, q, acc[t][1][k], 0, 0, 0);
          }
      }
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int w = 0; w < 2; w++) {
          sc[t][w] = acc[t][w][kN - 1];
#pragma unroll
          for (int k = kN - 2; k >= 0; k--) sc[t][w] += acc[t][w][k];
        }
    }
    if (more) load_k(next);

    uint32_t nan[2];
    float kscale[2], vscale[2];
    int first[2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
      const bool ok = cur[w].id >= 0;
      nan[w] = ok ? Meta::nan(cur[w].meta) : cur[w].id == -2 ? 0xffffu : 0u;
      kscale[w] = scale * pow2(ok ? Meta::ek(cur[w].meta) : 0);
      vscale[w] = pow2(ok ? Meta::ev(cur[w].meta) : 0);
      // (a page of no index lies behind every position)
      first[w] = cur[w].index >= 0 ? cur[w].index * kPage + 4 * kq : INT_MAX - kPage;
      if (!ok)
#pragma unroll
        for (int s = 0; s < kSegs; s++) vc[w][s] = u4{0, 0, 0, 0};
    }
    b8 wt[NT][kW];
#pragma unroll
    for (int t = 0; t < NT; t++) {
      float x[8];
#pragma unroll
      for (int w = 0; w < 2; w++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          x[4 * w + i] = first[w] + i < lim[t] ? sc[t][w][i] * kscale[w] : -INFINITY;
      if (nan[0] | nan[1]) {
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (first[w] + i < lim[t] && (nan[w] >> (4 * kq + i) & 1)) x[4 * w + i] = NAN;
      }
      float top = x[0];
#pragma unroll
      for (int i = 1; i < 8; i++) top = fmaxf(top, x[i]);
      top = fmaxf(m[t], quads_max(top));
      if (__any(top > m[t])) {
        const float down = top > -INFINITY ? __builtin_amdgcn_exp2f(m[t] - top) : 1.0f;
        l[t] *= down;
#pragma unroll
        for (int i = 0; i < kTiles; i++) o[t][i] *= down;
        m[t] = top;
      }
      const float at = top > -INFINITY ? top : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        x[i] = __builtin_amdgcn_exp2f(x[i] - at);
        l[t] += x[i];
        x[i] *= vscale[i / 4];
      }
      split_near<T>(x, wt[t]);
    }
#pragma unroll
    for (int s = 0; s < kSegs; s++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const b8 a = of_codes8(vc[0][s][i], vc[1][s][i]);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
          for (int k = kW - 1; k >= 0; k--)
            o[t][4 * s + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, wt[t][k], o[t][4 * s + i], 0, 0, 0);
      }
    if (more) {
      load_v(next);
      cur[0] = next[0];
      cur[1] = next[1];
    }
  }

  // the four waves' states, joined in wave order
#pragma unroll
  for (int t = 0; t < NT; t++) {
    l[t] = quads_sum(l[t]);
    if (kq == 0) lds_ml[wave][t * 16 + n16] = f2{m[t], l[t]};
  }
  const Partials part = partials_at<HD>(ws, slots, kQueries);
#pragma unroll
  for (int t = 0; t < NT; t++) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTiles; i++) reinterpret_cast<f4*>(lds)[(wave * kTiles + i) * 64 + lane] = o[t][i];
    __syncthreads();
    const int q = t * 16 + n16, qi = tile * kQueries + q;
    if (qi < nrows * group) {
      float top = -INFINITY, sum = 0, by[4];
#pragma unroll
      for (int w = 0; w < 4; w++) top = fmaxf(top, lds_ml[w][q][0]);
#pragma unroll
      for (int w = 0; w < 4; w++) {
        by[w] = lds_ml[w][q][0] > -INFINITY ? __builtin_amdgcn_exp2f(lds_ml[w][q][0] - top) : 1.0f;
        sum += by[w] * lds_ml[w][q][1];
      }
      const int row = row0 + qi / group, col = (head * group + qi % group) * HD;
      const float inv = sum == 0 ? 0.0f : 1.0f / sum;  // (nothing attended: zero)
      if (slot >= 0 && wave == 0 && kq == 0) part.ml[(int64_t)slot * kQueries + q] = f2{top, sum};
      for (int i = wave; i < kTiles; i += 4) {
        f4 x = reinterpret_cast<const f4*>(lds)[i * 64 + lane] * by[0];
#pragma unroll
        for (int w = 1; w < 4; w++) x += reinterpret_cast<const f4*>(lds)[(w * kTiles + i) * 64 + lane] * by[w];
        if (slot >= 0) *reinterpret_cast<f4*>(part.o + ((int64_t)slot * kQueries + q) * HD + i * 16 + kq * 4) = x;
        else store4<T>(out, row, col + i * 16 + kq * 4, x * inv);
      }
    }
  }
}

// ---- joining the chunks ---------------------------------------------------------------

// A wave per (row, head): the partial sums of its chunks in order.
template <int HD, int T, int NT, bool LIST>
__global__ __launch_bounds__(256) void merge_kernel(Rows r, Out out, List list, int kv_heads, void* ws, int slots) {
  constexpr int kQueries = 16 * NT, kLanes = HD / 4;  // lanes with 4 dims each
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int row = __builtin_amdgcn_readfirstlane((int)(id / r.heads)), h = __builtin_amdgcn_readfirstlane((int)(id % r.heads));
  if (row >= r.rows) return;
  const int group = r.heads / kv_heads, head = h / group;
  int chunks, slot, step, q;
  if constexpr (LIST) {
    const int seq = seq_of(r, row);
    if (seq < 0) return;
    const int count = min(max(list.count[(int64_t)row * kv_heads + head], 0), list.top), tiles = (group + 15) / 16;
    chunks = chunks_of(count, list.chunk);
    q = h % group;
    slot = ((row * kv_heads + head) * tiles + q / 16) * list.chunks;
    step = 1;
    q %= 16;
  } else {
    Found f;
    if (!find<true>(r, kv_heads, group, kQueries, row, f)) return;
    chunks = chunks_of(f.s.pages, f.chunk);
    q = (row - f.s.row0) * group + h % group;
    slot = f.slot + head * f.s.tiles + q / kQueries;
    step = kv_heads * f.s.tiles;
    q %= kQueries;
  }
  if (chunks == 1 || slot < 0 || (int64_t)slot + (int64_t)(chunks - 1) * step >= slots) return;
  const Partials part = partials_at<HD>(ws, slots, kQueries);
  float top = -INFINITY;
  for (int c = lane; c < chunks; c += 64) top = fmaxf(top, part.ml[((int64_t)slot + (int64_t)c * step) * kQueries + q][0]);
  top = wave_max(top);
  float sum = 0;
  f4 x{0, 0, 0, 0};
  for (int c0 = 0; c0 < chunks; c0 += 64) {
    f2 ml{-INFINITY, 0};
    if (c0 + lane < chunks) ml = part.ml[((int64_t)slot + (int64_t)(c0 + lane) * step) * kQueries + q];
    const float by = ml[0] > -INFINITY ? __builtin_amdgcn_exp2f(ml[0] - top) : 1.0f;
    sum += by * ml[1];
    const int many = min(chunks - c0, 64);
    const float* from = part.o + (((int64_t)slot + (int64_t)c0 * step) * kQueries + q) * HD + (lane % kLanes) * 4;
#pragma unroll 8
    for (int c = 0; c < many; c++)
      x += *reinterpret_cast<const f4*>(from + (int64_t)c * step * kQueries * HD) *
           __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, by), c));
  }
  sum = wave_sum(sum);
  if (lane < kLanes) store4<T>(out, row, (int64_t)h * HD + lane * 4, x * (sum == 0 ? 0.0f : 1.0f / sum));
}

// ---- launches ---------------------------------------------------------------------------

// Tiles of `queries` over all rows, at most.
int64_t tiles_most(int group, int nseq, int rows, int queries) {
  return (int64_t)rows * group / queries + (nseq < rows ? nseq : rows);
}

struct Grid {
  int64_t items, slots;
};
Grid grid_of(const Layout& at, int heads, int nseq, int max_blocks, int rows, int queries) {
  const int64_t tiles = tiles_most(heads / at.kv_heads, nseq, rows, queries) * at.kv_heads;
  const int64_t cut = tiles * ((max_blocks + kMinChunk - 1) / kMinChunk);
  // contexts longer than a chunk of c pages make at most twice (all tiles' pages) / c items, the rest one each
  return Grid{cut < tiles + kItems ? cut : tiles + kItems, cut < 2 * kItems ? cut : 2 * kItems};
}

int sparse_chunk(const Layout& at, int heads, int rows, int top) {
  const int64_t all = (int64_t)rows * at.kv_heads * ((heads / at.kv_heads + 15) / 16) * top;
  const int64_t c = ((all + kItems - 1) / kItems + 7) & ~7ll;
  return (int)(c > kMinChunk ? (c < 1 << 20 ? c : 1 << 20) : kMinChunk);
}

template <int HD, int T, int NT, bool LIST>
void launch(const Pool& p, const Rows& r, const Out& o, const List& list, void* ws, int64_t items, int64_t slots,
            bool merge, hipStream_t s) {
  item_kernel<HD, T, NT, LIST><<<(unsigned)items, 256, 0, s>>>(p, r, o, list, ws, (int)slots);
  PGD_HIP(hipGetLastError());
  if (!merge) return;
  const int64_t waves = (int64_t)r.rows * r.heads;
  merge_kernel<HD, T, NT, LIST><<<(unsigned)((waves + 3) / 4), 256, 0, s>>>(r, o, list, p.at.kv_heads, ws, (int)slots);
  PGD_HIP(hipGetLastError());
}

template <int NT, bool LIST>
void launch_of(const Pool& p, const Rows& r, const Out& o, const List& list, void* ws, int64_t items, int64_t slots,
               bool merge, hipStream_t s) {
  auto go = [&](auto hd, auto type) {
    launch<decltype(hd)::value, decltype(type)::value, NT, LIST>(p, r, o, list, ws, items, slots, merge, s);
  };
  auto typed = [&](auto hd) {
    if (r.type == F32) go(hd, std::integral_constant<int, F32>());
    else if (r.type == F16) go(hd, std::integral_constant<int, F16>());
    else go(hd, std::integral_constant<int, BF16>());
  };
  if (p.at.hd == 64) typed(std::integral_constant<int, 64>());
  else if (p.at.hd == 128) typed(std::integral_constant<int, 128>());
  else typed(std::integral_constant<int, 256>());
}

size_t partial_bytes(const Layout& at, int64_t slots, int queries) { return (size_t)slots * queries * (at.hd + 2) * 4; }

}  // namespace

size_t attn_ws_bytes(const Layout& at, int heads, int nseq, int max_blocks, int rows) {
  return partial_bytes(at, grid_of(at, heads, nseq, max_blocks, rows, 16).slots, 16);
}

void attn(const Pool& p, const Rows& r, int max_rows, const Out& o, void* ws, hipStream_t s) {
  const Grid g = grid_of(p.at, r.heads, r.nseq, r.max_blocks, r.rows, 16);
  launch_of<1, false>(p, r, o, List{}, ws, g.items, g.slots, r.max_blocks > kMinChunk, s);
}

size_t attn_sparse_ws_bytes(const Layout& at, int heads, int rows, int top) {
  const int c = sparse_chunk(at, heads, rows, top), chunks = (top + c - 1) / c;
  if (chunks <= 1) return 0;
  return partial_bytes(at, (int64_t)rows * at.kv_heads * ((heads / at.kv_heads + 15) / 16) * chunks, 16);
}

void attn_sparse(const Pool& p, const Rows& r, int top, const int* sel, const int* count, const Out& o, void* ws,
                 hipStream_t s) {
  const int c = sparse_chunk(p.at, r.heads, r.rows, top), chunks = (top + c - 1) / c;
  const int64_t items = (int64_t)r.rows * p.at.kv_heads * ((r.heads / p.at.kv_heads + 15) / 16) * chunks;
  launch_of<1, true>(p, r, o, List{sel, count, top, c, chunks}, ws, items, items, chunks > 1, s);
}

}  // namespace kv8
}  // namespace pgd
