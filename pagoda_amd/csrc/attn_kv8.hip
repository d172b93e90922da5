// attn_kv8.hip — causal GQA attention over the 8-bit paged KV cache: all pages of a
// sequence, or per (row, KV head) the pages of a list.
//
// For a query q of a row at position p:  o = sum_j w_j v_j / sum_j w_j over j <= p,
// w_j = exp(q.k_j / sqrt(hd)), with k_j = 2^ek codes, v_j = 2^ev codes per page and head.
// Per two pages (32 positions) and a tile of 16 queries (rows x group heads):
//   S[pos][query]  = K codes . q        16x16x32 f16 products over hd / 32 steps
//   t = S 2^ek log2(e) / sqrt(hd), its running maximum m and the sum l of 2^(t - m) in f32
//   O[dim][query] += V codes^T . 2^(t - m + ev - d)   the same products over the 32 positions
// with d the running maximum of t - m + ev, rounded up, so that the largest weight of a value's code is
// about one whatever the pages' powers of two (both maxima may lag behind, m a factor of 2^4 and d one of 2^3). d is a
// whole number near the pages' exponents: adding them to it and taking it back from results is exact, also where
// scores are so large that t + ev would not be.
// Codes convert to f16 exactly. Queries are scaled by a power of two into f16's range and enter as f16 terms: f32
// rows two (22 bits), f16 rows themselves, bf16 rows one (exact): all to half of f16's smallest step, 2^-25 where the
// largest entry is 2^14 or more. The weights, times 2^12, enter as two terms, 2^-21, and 2^-36 of the largest. With one
// term, an eighth of bf16's own rounding, up to one bf16 result in 200 is a neighbour of the exact one's rounding. bf16
// terms would need no scaling but half as many more products: three for f32 where f16 takes two.
// The lane that holds a score holds it as the operand of the second product: lane
// (query n = l % 16, kq = l / 16) has positions 4 kq .. 4 kq + 3 of both pages, which
// are the 8 that a lane of the second product's operand takes, and its results are
// columns n too, so m, d, l and the rescaling stay in the lane but for two maxima
// over the four kq.
//
// Split: work is a list of (sequence, chunk of pages, KV head, tile of queries) that every
// workgroup derives for itself from the row starts and lengths on the device, so a call
// needs no plan from the host. Sequences of few queries take item_kernel: tiles of 16
// queries, four waves on pairs of pages in turn, each with its own maxima, sum and O, joined
// in LDS. The others take prompt_kernel: the four waves of a workgroup have
// queries of their own and walk the same pages, staged in LDS for all. Contexts of one chunk
// write results, the others partial sums that merge_kernel adds in chunk order.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "kv8_dev.h"

namespace pgd {
namespace kv8 {

namespace {

// Items that contexts are cut into, about. item_kernel: as many as run at once (workgroups of four waves that a
// CU holds at a head_dim, over the 256 CUs).
constexpr int few_items(int hd, int tiles) { return 256 * (hd == 256 ? 2 : hd == 128 ? 3 : 4) / tiles; }
constexpr int many_items(int hd) { return hd == 128 ? 1024 : 1536; }
// prompt_kernel: more, as contexts that are cut or not make uneven rounds (3 prompts of 2274 rows, head_dim 256: 277 us
// against 346 with 512 items), but as many as run at once rather than chunks of less than kFullChunk pages, which the
// way to their first page and their partial sums would make dear (236 rows on 3977 positions, head_dim 256: 74 us
// against 97; 30 on 15000: 49 against 81; 500 on 3977: 122 against 130; with 32 pages 82, 49 and 131; but two prompts of
// 1500 rows on 900 and 3000 at head_dim 64: 64 against 62).
constexpr int many_at_once(int hd) { return hd == 64 ? 1024 : 512; }
constexpr int kFullChunk = 64;
constexpr int kMinChunk = 8;     // pages: a pair for each of four waves
constexpr int kOneChunk = 16;    // pages of tables (and lists) that are never cut: the join would cost more
// Queries of a sequence and KV head: calls of up to these are item_kernel's alone. 16 sequences of 100 to 6000
// positions, 7 queries a row at head_dim 64 (f32) and 128 (bf16), 6 at 256 (f16), with this and with 32: at 64 12 rows
// each 20 and 31 us, 18 rows 23 and 33; at 128 8 rows 31 and 34, 12 rows 38 and 41, but 18 rows 45 and 42; at 256 12 rows
// 57 and 59, 1 to 20 rows 46 and 54, but 20 rows 66 and 63. 30 rows (past both) the same.
constexpr int kFewQueries = 128;

template <int T>
constexpr int kTerms = T == F32 ? 2 : 1;  // f16 terms of a query
constexpr int kWeightTerms = 2;
// O and the sum are only brought to new maxima that are 2^kSlack (of weights) or 2^kSlackV (of weights of codes) times
// the old ones or more (and all of a wave's with them), so weights of codes reach 2^kSlackV. They enter times
// 2^kWeightExp: f16 holds 2^-24 to 65504.
constexpr float kSlack = 4, kSlackV = 3, kWeightExp = 15 - kSlackV;
constexpr float kLowest = -3.402823466e38f;

// x as f16 terms to nearest, each of what the ones before leave.
template <int N>
__device__ inline void split(const float (&x)[8], h8 (&out)[N]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; j++) r[j] = x[j];
#pragma unroll
  for (int k = 0; k < N; k++) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
      out[k][j] = (_Float16)r[j];
      if (k + 1 < N) r[j] -= (float)out[k][j];
    }
  }
}

// The same for weights, in fewer instructions: all terms but the last truncated, two at a time (what is left is
// exact), the last to nearest.
template <int N>
__device__ inline void split_weights(const float (&x)[8], h8 (&out)[N]) {
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; j++) r[j] = x[j];
#pragma unroll
  for (int k = 0; k < N; k++)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if (k + 1 < N) {
        const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(r[j], r[j + 1]));
        out[k][j] = h[0];
        out[k][j + 1] = h[1];
        r[j] -= (float)h[0];
        r[j + 1] -= (float)h[1];
      } else {
        out[k][j] = (_Float16)r[j];
        out[k][j + 1] = (_Float16)r[j + 1];
      }
    }
}

// Eight codes as f16.
__device__ inline h8 of_codes8(uint32_t lo, uint32_t hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
  const h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
  const h2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ---- the list of items ------------------------------------------------------------

struct Seq {
  int row0, n;      // its rows
  int len;          // positions as given
  int ctx, pages;   // positions that the table holds, and their pages
};

__device__ inline Seq seq_at(const Rows& r, int i) {
  Seq s;
  const int a = min(max(r.row_start[i], 0), r.rows), b = min(max(r.row_start[i + 1], 0), r.rows);
  s.row0 = a;
  s.n = max(b - a, 0);
  s.len = r.lens[i];
  const long long most = (long long)r.max_blocks * kPage;
  s.ctx = (int)min((long long)max(s.len, 0), most);
  s.pages = (s.ctx + kPage - 1) / kPage;
  return s;
}

// A kernel's share of a call: sequences of at least `least` and at most `most` queries a KV head, in tiles.
struct Share {
  int least, most;
  int tile;   // queries, a power of two
  int items;  // that contexts are cut into, about
  int fewest;  // as many, rather than chunks of less than kFullChunk pages
};

struct Class {
  int group;
  Share sh;
  __device__ int tiles(int n) const {
    const int q = n * group;  // (rows * heads stay below 2^26)
    return q < sh.least || q > sh.most ? 0 : (q + sh.tile - 1) >> __builtin_ctz(sh.tile);
  }
  // partial sums are of 16 queries, whatever the tile
  __device__ int tiles16(int n) const { return (n * group + 15) >> 4; }
};

// The workspace's partial sums: how many it has, and a launch's own.
struct Slots {
  int all, first, end;
};

__device__ inline int chunks_of(int pages, int chunk) { return pages > 0 ? (pages + chunk - 1) / chunk : 1; }

__device__ __host__ inline int least_chunk(int max_blocks) { return max_blocks <= kOneChunk ? kOneChunk : kMinChunk; }

// Pages of a chunk of a context, where all contexts' tiles together are to be cut into chunks of about `each`
// pages: contexts are cut evenly, into multiples of 8 pages (a pair for each of four waves).
__device__ inline int chunk_of(int pages, float each, int least) {
  const float n = fmaxf(floorf((float)pages / each + 0.25f), 1.0f);
  return max(((int)ceilf((float)pages / n) + 7) & ~7, least);
}

struct Found {
  Seq s;
  int seq, tiles, chunk;
  int local;  // the item among the sequence's
  int slot;   // the sequence's first partial sum
};

// The sequence of a workgroup's item, as every wave works it out for itself, 64 sequences at a time.
// Returns false for the workgroups past the list.
__device__ inline bool find(const Rows& r, int kv_heads, const Class& cl, int key, Found& f) {
  const int lane = threadIdx.x & 63;
  const bool strip = r.nseq <= 64;  // one strip: nothing is loaded twice
  Seq s{};
  int tiles = 0;
  float all = 0;
  for (int base = 0; base < r.nseq; base += 64) {
    const int i = base + lane;
    tiles = 0;
    if (i < r.nseq) {
      s = seq_at(r, i);
      tiles = cl.tiles(s.n);
    }
    all += (float)tiles * (float)s.pages;
  }
  const float total = wave_total(all) * kv_heads;
  const float each = fmaxf(fmaxf(total / cl.sh.items, fminf(total / cl.sh.fewest, kFullChunk)), 1.0f);
  const int least = least_chunk(r.max_blocks);
  int chunk = 0;  // this lane's sequence's
  auto items_of = [&](int base) {
    if (!strip) {
      tiles = 0;
      if (base + lane < r.nseq) {
        s = seq_at(r, base + lane);
        tiles = cl.tiles(s.n);
      }
    }
    chunk = chunk_of(s.pages, each, least);
    return tiles * chunks_of(s.pages, chunk) * kv_heads;
  };
  int before = 0, split_before = 0;
  for (int base = 0; base < r.nseq; base += 64) {
    const int mine = items_of(base), upto = before + wave_scan(mine);
    const int chunks = chunks_of(s.pages, chunk);
    const int slots = chunks > 1 && tiles > 0 ? cl.tiles16(s.n) * kv_heads * chunks : 0;
    const int slots_upto = split_before + wave_scan(slots);
    const uint64_t hit = __ballot(key < upto && key >= upto - mine);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      f.s.row0 = __builtin_amdgcn_readlane(s.row0, src);
      f.s.n = __builtin_amdgcn_readlane(s.n, src);
      f.s.len = __builtin_amdgcn_readlane(s.len, src);
      f.s.ctx = __builtin_amdgcn_readlane(s.ctx, src);
      f.s.pages = __builtin_amdgcn_readlane(s.pages, src);
      f.tiles = __builtin_amdgcn_readlane(tiles, src);
      f.chunk = __builtin_amdgcn_readlane(chunk, src);
      f.local = key - __builtin_amdgcn_readlane(upto - mine, src);
      f.slot = __builtin_amdgcn_readlane(slots_upto - slots, src);
      f.seq = base + src;
      return true;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
    split_before = __builtin_amdgcn_readlane(slots_upto, 63);
  }
  return false;
}

// Positions that row j of a sequence sees.
__device__ inline int seen_by(const Seq& s, int j) {
  return (int)max(min((long long)s.len - s.n + j + 1, (long long)s.ctx), 0ll);
}

// Pages that the last row of a tile sees.
__device__ inline int tile_pages(const Seq& s, int group, int tile_queries, int tile) {
  const int last = min(((tile + 1) * tile_queries - 1) / group, s.n - 1);
  return (seen_by(s, last) + kPage - 1) / kPage;
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
    for (int j = 0; j < 4; j++) x[j] /= 1.0f + __builtin_amdgcn_exp2f(g[j] * -1.44269504088896f);
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

// What merge_kernel needs to know of a row's sequence, left by the first item of the row's tile.
struct RowPart {
  int slot, chunk, row0, n, len, tile_queries, pad[2];
};

// Workspace: RowPart of every row, then per slot (16 queries of a chunk and head) O [16][hd], then their
// (m, d, l).
struct Partials {
  RowPart* rows;
  float* o;
  f4* st;
};
template <int HD>
__device__ __host__ inline Partials partials_at(void* ws, int rows, int slots) {
  Partials p;
  p.rows = static_cast<RowPart*>(ws);
  p.o = reinterpret_cast<float*>(p.rows + rows);
  p.st = reinterpret_cast<f4*>(p.o + (size_t)slots * 16 * HD);
  return p;
}

// What several runs over parts of a context leave, joined: maxima and the sum.
struct State {
  float m = -INFINITY, d = -INFINITY, l = 0;
  // d of a part, from m on (-infinity of one that attended nothing).
  __device__ float level(f4 s) const { return s[0] > -INFINITY ? ceilf(s[0] - m + s[1]) : -INFINITY; }
  // The factor of a part's O (a part that attended nothing has zeros, or NaN, to keep).
  __device__ float of_part(f4 s) const { return s[0] > -INFINITY ? __builtin_amdgcn_exp2f((s[0] - m) + (s[1] - d)) : 1.0f; }
  __device__ float sum_of_part(f4 s) const { return (s[0] > -INFINITY ? __builtin_amdgcn_exp2f(s[0] - m) : 1.0f) * s[2]; }
  template <int N, class F>
  __device__ void join(F part, float (&by)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) m = fmaxf(m, part(i)[0]);
#pragma unroll
    for (int i = 0; i < N; i++) d = fmaxf(d, level(part(i)));
#pragma unroll
    for (int i = 0; i < N; i++) by[i] = of_part(part(i)), l += sum_of_part(part(i));
  }
  // O to results, x * by * 2^exp: the power of two may lie below the normal range where the result does not. Nothing
  // attended gives zero.
  struct Factor {
    float by;
    int exp;
    __device__ f4 operator()(f4 x) const {
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = __builtin_ldexpf(x[i] * by, exp);
      return x;
    }
  };
  __device__ Factor factor() const {
    if (l == 0) return Factor{0.0f, 0};
    if (m == kLowest) return Factor{NAN, 0};  // all scores lie below f32's range, who knows how far apart
    return Factor{1.0f / l, d > -INFINITY ? (int)(d - kWeightExp) : 0};
  }
};

struct List {
  const int *sel, *count;
  int top, chunk, chunks;  // pages of a chunk and chunks of a full list
};

// The RowParts of the rows whose first query a tile has.
__device__ inline void leave_row_parts(const Partials& part, const Seq& s, int group, int tile, int tile_queries,
                                       const Found& f, const Slots& slots) {
  const int j = (tile * tile_queries + group - 1) / group + (int)threadIdx.x;
  if ((int)threadIdx.x < tile_queries && j < s.n && j * group < (tile + 1) * tile_queries)
    part.rows[s.row0 + j] = RowPart{slots.first + f.slot, f.chunk, s.row0, s.n, s.len, tile_queries, {0, 0}};
}

// ---- 16 queries and two pages ---------------------------------------------------------

// The next 64 pages of a walk, one a lane: places in the table and page numbers.
// number: -1 for no page, -2 for one outside the pool (attending it makes NaN).
struct Walk {
  int index = -1, id = -1;
  __device__ void set(int at, const int* table, int max_blocks, int n_pages) {
    index = at;
    id = -1;
    if (at >= 0 && at < max_blocks) {
      const int p = table[at];
      id = p >= 0 && p < n_pages ? p : -2;
    } else {
      index = -1;
    }
  }
};

struct Page {
  int index, id;
  uint32_t meta;
  const uint8_t* at;
};

struct PoolAt {
  const uint8_t* base;
  size_t page_bytes, head, meta;
  __device__ PoolAt(const Pool& p, int h)
      : base(p.base), page_bytes(p.at.page_bytes()), head((size_t)h * p.at.head_bytes()), meta(p.at.meta_at() + (size_t)h * 4) {}
  __device__ Page page(const Walk& w, int lane) const {
    Page g;
    g.index = __builtin_amdgcn_readlane(w.index, lane);
    g.id = __builtin_amdgcn_readlane(w.id, lane);
    const uint8_t* p = base + (size_t)max(g.id, 0) * page_bytes;
    g.at = p + head;
    g.meta = *reinterpret_cast<const uint32_t*>(p + meta);
    return g;
  }
};

// A query's running maxima, sum (of this lane's positions) and scaling, as its column of lanes holds them.
struct Query {
  float m = -INFINITY, d = -INFINITY, l = 0;
  int exp = 0, lim = 0;  // power of two of its terms; positions it sees
};

// Scores of PG pages' positions to weights: s[w][i] is position 16 index + 4 kq + i of page w.
template <int PG, int N>
__device__ inline void weigh(const f4 (&s)[PG], const Page (&pg)[PG], float scale, bool whole, Query& q, f4 (&o)[N],
                             h8 (&out)[PG / 2][kWeightTerms]) {
  const int kq = threadIdx.x >> 4 & 3;
  float x[PG][4], by[PG], ev[PG];
  int ek[PG], highest = INT_MIN;
#pragma unroll
  for (int w = 0; w < PG; w++) {
    // (for no page the pool's first one was loaded: what that holds must not show, be it in the rounding of results)
    const uint32_t meta = pg[w].id >= 0 ? pg[w].meta : Meta::pack(kExpMin, kExpMin, 0);
    ek[w] = Meta::ek(meta);
    ev[w] = (float)Meta::ev(meta);
    // (not below the normal range: the scores of masked positions are infinite)
    by[w] = fmaxf(__builtin_ldexpf(scale, q.exp + ek[w]), 1.17549435e-38f);
    highest = max(highest, ek[w]);
#pragma unroll
    for (int i = 0; i < 4; i++) x[w][i] = s[w][i];
  }
  if (__any(q.exp + highest > 96)) {
    // (s stays below 2^33.) The factor may be infinite where keys and queries have no channel in common, so its power of
    // two comes last. A score below f32's range becomes its lowest number: -infinity is a masked position's.
#pragma unroll
    for (int w = 0; w < PG; w++) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float t = __builtin_ldexpf(x[w][i] * scale, q.exp + ek[w]);
        x[w][i] = t < kLowest ? kLowest : t;
      }
      by[w] = 1.0f;
    }
  }
  if (!whole) {
#pragma unroll
    for (int w = 0; w < PG; w++) {
      const uint32_t nan = pg[w].id >= 0 ? Meta::nan(pg[w].meta) : pg[w].id == -2 ? 0xffffu : 0u;
      // (a page of no index lies behind every position)
      const int first = pg[w].index >= 0 ? pg[w].index * kPage + 4 * kq : INT_MAX - kPage;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float v = nan >> (4 * kq + i) & 1 ? NAN : x[w][i];
        x[w][i] = first + i < q.lim ? v : -INFINITY;
      }
    }
  }
  // This lane's largest t and t - m + ev. What its column's other lanes have need not be known while no lane of the
  // wave is past what its column's maxima may lag.
  auto largest = [&](int w) { return fmaxf(fmaxf(x[w][0], x[w][1]), fmaxf(x[w][2], x[w][3])) * by[w]; };
  float top = -INFINITY, top_v = -INFINITY;
#pragma unroll
  for (int w = 0; w < PG; w++) {
    const float t = largest(w);
    top = fmaxf(top, t);
    top_v = fmaxf(top_v, t - q.m + ev[w]);
  }
  if (__any(top > q.m + kSlack || top_v > q.d + kSlackV)) {
    const float m = fmaxf(q.m, quads_max(top)), base = m > -INFINITY ? m : 0.0f;
    top_v = -INFINITY;
#pragma unroll
    for (int w = 0; w < PG; w++) top_v = fmaxf(top_v, largest(w) - base + ev[w]);
    const float d = ceilf(fmaxf(quads_max(top_v), q.d + (q.m - base)));
    if (q.m > -INFINITY) {  // (else O holds zeros, or NaN)
      q.l *= __builtin_amdgcn_exp2f(q.m - base);
      const float down = __builtin_amdgcn_exp2f((q.m - base) + (q.d - d));
#pragma unroll
      for (int i = 0; i < N; i++) o[i] *= down;
    }
    q.m = m;
    q.d = d;
  }
  const float at = q.m > -INFINITY ? q.m : 0.0f, up = q.d > -INFINITY ? kWeightExp - q.d : 0.0f;
  if (__any(fabsf(at) > 65536.0f)) {
    // m is a rounded product: an exact one would lie past it by up to its half step, which may be many powers of two
#pragma unroll
    for (int w = 0; w < PG; w++) {
#pragma unroll
      for (int i = 0; i < 4; i++) x[w][i] *= by[w];
      by[w] = 1.0f;
    }
  }
  float far = -INFINITY, sum[PG];
#pragma unroll
  for (int w = 0; w < PG; w++) far = fmaxf(far, ev[w]);
  const bool apart = __any(up + far > 100.0f);
#pragma unroll
  for (int w = 0; w < PG; w++) {
    const float f = up + ev[w];
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x[w][i] = __builtin_fmaf(x[w][i], by[w], -at);
#pragma unroll
    for (int i = 0; i < 4; i++) e[i] = __builtin_amdgcn_exp2f(x[w][i]);
    sum[w] = (e[0] + e[1]) + (e[2] + e[3]);
    if (apart) {
      // pages so far apart that 2^(t - m) underflows where the weight does not
#pragma unroll
      for (int i = 0; i < 4; i++) x[w][i] = __builtin_amdgcn_exp2f(x[w][i] + f);
    } else {
      const float of_code = __builtin_amdgcn_exp2f(f);
#pragma unroll
      for (int i = 0; i < 4; i++) x[w][i] = e[i] * of_code;
    }
  }
#pragma unroll
  for (int w = 0; w < PG; w++) q.l += sum[w];
#pragma unroll
  for (int w = 0; w < PG; w += 2) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = x[w + i / 4][i & 3];
    split_weights(v, out[w / 2]);
  }
}

// Whether all of some pages' positions count for every query of a wave that sees at least `least`.
template <int PG>
__device__ inline bool whole_pages(const Page (&pg)[PG], int least) {
  bool whole = true;
#pragma unroll
  for (int w = 0; w < PG; w++)
    whole &= pg[w].id >= 0 && Meta::nan(pg[w].meta) == 0 && (pg[w].index + 1) * kPage <= least;
  return whole;
}

// Eight dims of a query as f16 terms; x is scaled to [2^14, 2^15) for the largest magnitude (below 2^-126: by 2^141) of
// the HD / 8 lanes that hold the query. Returns the power of two it was divided by.
template <int T, int HD, int N>
__device__ inline int query_terms(float (&x)[8], h8 (&t)[N]) {
  // An infinity becomes NaN: scores of -infinity alone would be those of masked positions.
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = __builtin_fmaf(x[j], 0.0f, x[j]);
  int e = 0;
  if constexpr (T != F16) {
    float most = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) most = fmaxf(most, fabsf(x[j]));
    most = lanes_max<HD / 8>(most);
    e = (int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127 - 14;
    // (2^-e may lie past f32: two powers of two)
    const float up = pow2(min(-e, 126)), more = pow2(max(-e - 126, 0));
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = x[j] * up * more;
  }
  split<N>(x, t);
  return e;
}

// ---- few queries a sequence ------------------------------------------------------------

// NQ tiles of 16 queries, four waves each, side by side over the same pages: what one loads the other finds in the
// caches. Bound by HBM at long contexts (8 of 20000 to 130000 positions, 4 heads of 128, bf16: 98 us, 5.1 TB/s); at
// short ones 5 us of the chain from row starts to pages go before it (32 of 40 to 4000, 4 heads of 256, f32: 18.8 us,
// 3.2 TB/s).
template <int HD, int T, int NQ, bool LIST>
__global__ __launch_bounds__(256 * NQ, 2) void item_kernel(Pool p, Rows r, Out out, List list, Share share, void* ws,
                                                           Slots slots) {
  constexpr int kSegs = HD / 64, kSteps = HD / 32, kTiles = HD / 16, kN = kTerms<T>, kW = kWeightTerms;
  constexpr int kJoinTiles = kTiles < 8 ? kTiles : 8;  // tiles of O joined at a time
  constexpr int kQBytes = kN * kSteps * 1024, kJoinBytes = 4 * kJoinTiles * 1024;
  constexpr int kTileBytes = kQBytes > kJoinBytes ? kQBytes : kJoinBytes;
  constexpr int kUnits = 16 * HD / 8;  // of 8 dims of a query
  constexpr int kRounds = kUnits > 256 ? kUnits / 256 : 1;
  __shared__ __align__(16) uint8_t lds_all[NQ * kTileBytes];
  __shared__ f4 lds_st_all[NQ][4][16];
  __shared__ int lds_exp_all[NQ][16];  // of the queries' powers of two
  const int sub = NQ > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  const int tid = threadIdx.x & 255, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint8_t* const lds = lds_all + sub * kTileBytes;
  f4(*const lds_st)[16] = lds_st_all[sub];
  int* const lds_exp = lds_exp_all[sub];
  const int n16 = lane & 15, kq = lane >> 4;
  const int kv_heads = p.at.kv_heads, group = r.heads / kv_heads;
  const Partials part = partials_at<HD>(ws, LIST ? 0 : r.rows, slots.all);

  // This wave's pairs are pages page0 + 2 (wave + 4 it) and the next.
  auto nth = [&](int it) { return 2 * (wave + 4 * (it + (lane >> 1))) + (lane & 1); };
  float x[kRounds][8];
  auto load_q = [&](const Seq& s, int head, int tile) {
#pragma unroll
    for (int i = 0; i < kRounds; i++) {
      const int u = tid + i * 256, qi = tile * 16 + u / (HD / 8);
#pragma unroll
      for (int j = 0; j < 8; j++) x[i][j] = 0;
      if (u < kUnits && qi < s.n * group)
        load8<T>(r.q, (int64_t)(s.row0 + qi / group) * r.ldq + (head * group + qi % group) * HD + u % (HD / 8) * 8, x[i]);
    }
  };

  // which pages, head and queries
  Seq s;
  int seq, head, tile, page0, page1, slot;
  int listed = -1;  // LIST: this lane's first page of the list
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
    // what needs no other load is on its way together
    page0 = c * list.chunk;
    pages_list = list.sel + ((int64_t)row * kv_heads + head) * list.top;
    if (nth(0) < list.chunk && page0 + nth(0) < list.top) listed = pages_list[page0 + nth(0)];
    s.row0 = row;
    s.n = 1;
    load_q(s, head, tile);
    const int count = min(max(list.count[(int64_t)row * kv_heads + head], 0), list.top);
    const RowSeq rs = row_seq(r, row);
    seq = rs.seq;
    const int have = chunks_of(count, list.chunk);
    if (c >= have || seq < 0) return;
    page1 = min(page0 + list.chunk, count);
    // (as the last of the rows up to this one)
    s.len = rs.seen(row);
    s.ctx = (int)min((long long)s.len, (long long)r.max_blocks * kPage);
    s.pages = (s.ctx + kPage - 1) / kPage;
    slot = have > 1 ? (int)blockIdx.x : -1;
  } else {
    Found f;
    const Class cl{group, share};
    if (!find(r, kv_heads, cl, blockIdx.x, f)) return;
    s = f.s;
    seq = f.seq;
    int local = f.local;
    const int tile_of = local % f.tiles;
    local /= f.tiles;
    head = local % kv_heads;
    const int c = local / kv_heads, pages = tile_pages(s, group, 16 * NQ, tile_of), have = chunks_of(pages, f.chunk);
    if (c == 0 && head == 0 && slots.all > 0) leave_row_parts(part, s, group, tile_of, share.tile, f, slots);
    if (c >= have) return;
    page0 = c * f.chunk;
    page1 = min(page0 + f.chunk, pages);
    tile = tile_of * NQ + sub;
    slot = have > 1 ? slots.first + f.slot + (c * kv_heads + head) * cl.tiles16(s.n) + tile : -1;
    if (slot >= slots.end) slot = INT_MAX;  // (row starts that do not ascend)
  }
  const int* table = r.block_tables + (int64_t)seq * r.max_blocks;

  const int pairs = (page1 - page0 - 2 * wave + 7) / 8;
  Walk walk;
  auto refill = [&](int it) {
    const int i = page0 + nth(it);
    int at = -1;
    if (i < page1) at = !LIST ? i : it == 0 ? listed : pages_list[i];
    // (what the table says past a row's context, and what such pages hold, may be anything)
    walk.set(at, table, LIST ? s.pages : r.max_blocks, p.n_pages);
  };
  if (pairs > 0) refill(0);
  if constexpr (!LIST) load_q(s, head, tile);
  const PoolAt pool(p, head);
  u4 kc[2][kSegs], vc[2][kSegs];
  auto load_k = [&](const Page (&g)[2]) {
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int i = 0; i < kSegs; i++) kc[w][i] = reinterpret_cast<const u4*>(g[w].at)[i * 64 + lane];
  };
  auto load_v = [&](const Page (&g)[2]) {
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int i = 0; i < kSegs; i++) vc[w][i] = reinterpret_cast<const u4*>(g[w].at + kPage * HD)[i * 64 + lane];
  };
  Page cur[2], next[2];
  if (pairs > 0) {
    cur[0] = pool.page(walk, 0);
    cur[1] = pool.page(walk, 1);
    load_k(cur);
    load_v(cur);
  }

  // the tile's queries as operands: per (term, step) lane l's 16 bytes at 16 l
#pragma unroll
  for (int i = 0; i < kRounds; i++) {
    const int u = tid + i * 256, g8 = u % (HD / 8), q = u / (HD / 8);
    h8 t[kN] = {};
    int e = 0;
    if (tile * 16 + i * 256 / (HD / 8) < s.n * group) e = query_terms<T, HD>(x[i], t);  // (any live query among them)
    if (u < kUnits) {
      if (g8 == 0) lds_exp[q] = e;
      // dims 64 seg + 16 kq + 8 half
      const int step = (g8 >> 3) * 2 + (g8 & 1), k4 = g8 >> 1 & 3;
#pragma unroll
      for (int k = 0; k < kN; k++) reinterpret_cast<h8*>(lds)[(k * kSteps + step) * 64 + k4 * 16 + q] = t[k];
    }
  }
  __syncthreads();

  const float scale = 1.44269504088896340736f / sqrtf((float)HD);
  const int qi = tile * 16 + n16;
  const bool live = qi < s.n * group;
  Query q;
  q.exp = lds_exp[n16];
  // (columns without a query, all zeros, go along with the last row)
  q.lim = seen_by(s, min(qi, s.n * group - 1) / group);
  const int least = seen_by(s, min(tile * 16, s.n * group - 1) / group);  // (rows see more and more)
  f4 o[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; i++) o[i] = f4{0, 0, 0, 0};

  for (int it = 0; it < pairs; it++) {
    const bool more = it + 1 < pairs;
    if (more) {
      if (((it + 1) & 31) == 0) refill(it + 1);
      next[0] = pool.page(walk, 2 * ((it + 1) & 31));
      next[1] = pool.page(walk, 2 * ((it + 1) & 31) + 1);
    }
    f4 sc[2] = {f4{0, 0, 0, 0}, f4{0, 0, 0, 0}};
#pragma unroll
    for (int step = 0; step < kSteps; step++) {
      const int i = step >> 1, h = step & 1;
      const h8 a0 = of_codes8(kc[0][i][2 * h], kc[0][i][2 * h + 1]);
      const h8 a1 = of_codes8(kc[1][i][2 * h], kc[1][i][2 * h + 1]);
#pragma unroll
      for (int k = 0; k < kN; k++) {
        const h8 b = reinterpret_cast<const h8*>(lds)[(k * kSteps + step) * 64 + lane];
        sc[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, b, sc[0], 0, 0, 0);
        sc[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, b, sc[1], 0, 0, 0);
      }
    }
    if (more) load_k(next);
#pragma unroll
    for (int w = 0; w < 2; w++)
      if (cur[w].id < 0)
#pragma unroll
        for (int i = 0; i < kSegs; i++) vc[w][i] = u4{0, 0, 0, 0};
    h8 wt[1][kW];
    weigh(sc, cur, scale, whole_pages(cur, least), q, o, wt);
#pragma unroll
    for (int i = 0; i < kSegs; i++) {
      h8 a[4];
#pragma unroll
      for (int j = 0; j < 4; j++) a[j] = of_codes8(vc[0][i][j], vc[1][i][j]);
      // (terms outermost: a product on the same sums as the one before it would wait for it)
#pragma unroll
      for (int k = kW - 1; k >= 0; k--)
#pragma unroll
        for (int j = 0; j < 4; j++)
          o[4 * i + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], wt[0][k], o[4 * i + j], 0, 0, 0);
    }
    if (more) {
      load_v(next);
      cur[0] = next[0];
      cur[1] = next[1];
    }
  }

  // the four waves' states, joined in wave order
  q.l = quads_sum(q.l);
  if (kq == 0) lds_st[wave][n16] = f4{q.m, q.d, q.l, 0};
  State st;
  State::Factor result{};
  float by[4];
#pragma unroll
  for (int t0 = 0; t0 < kTiles; t0 += kJoinTiles) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinTiles; i++) reinterpret_cast<f4*>(lds)[(wave * kJoinTiles + i) * 64 + lane] = o[t0 + i];
    __syncthreads();
    if (t0 == 0) {
      st.join<4>([&](int w) { return lds_st[w][n16]; }, by);
      result = st.factor();
      if (live && slot >= 0 && slot < INT_MAX && wave == 0 && kq == 0) part.st[(int64_t)slot * 16 + n16] = f4{st.m, st.d, st.l, 0};
    }
    if (live) {
      const int row = s.row0 + qi / group, col = (head * group + qi % group) * HD;
#pragma unroll 1
      for (int i = wave; i < kJoinTiles; i += 4) {
        f4 v = reinterpret_cast<const f4*>(lds)[i * 64 + lane] * by[0];
#pragma unroll
        for (int w = 1; w < 4; w++) v += reinterpret_cast<const f4*>(lds)[(w * kJoinTiles + i) * 64 + lane] * by[w];
        const int d = (t0 + i) * 16 + kq * 4;
        if (slot == INT_MAX) continue;
        if (slot >= 0) *reinterpret_cast<f4*>(part.o + ((int64_t)slot * 16 + n16) * HD + d) = v;
        else store4<T>(out, row, col + d, result(v));
      }
    }
  }
}

// ---- many queries a sequence -------------------------------------------------------------

// Workgroup: 64 queries, 16 a wave, over the pages of a chunk, PG at a time through LDS (two buffers, one
// barrier a step). A wave keeps its queries' terms in registers. 32 queries a wave would share the codes' conversion
// and measured slower, with fewer waves (1500 bf16 rows on 3900 positions at head_dim 128 107 against 91 us, with one
// term of weights; with two this form takes 97).
// Bound by issue: 5 VALU instructions (codes to f16, softmax) for each matrix instruction of 16 clocks, which are busy
// 37% of the time. 2274 f32 rows on 500 to 4001 positions, 24 / 4 heads of 256: 174 to 330 us by how rows fall on
// contexts. 1000 bf16 rows on 4000 positions 206 us.
template <int HD, int T, int PG>
__global__ __launch_bounds__(256, 2) void prompt_kernel(Pool p, Rows r, Out out, Share share, void* ws, Slots slots) {
  constexpr int kSegs = HD / 64, kSteps = HD / 32, kTiles = HD / 16, kN = kTerms<T>, kW = kWeightTerms;
  constexpr int kHead = 2 * kPage * HD;            // bytes of a page and head
  constexpr int kRounds = PG * kHead / 4096;       // 16 bytes a thread each, of a step
  constexpr int kQueries = 64;
  constexpr int kQBytes = 16 * HD * 2;             // 16 queries' operands of one term
  constexpr int kLds = 2 * PG * kHead > 4 * kQBytes ? 2 * PG * kHead : 4 * kQBytes;
  __shared__ __align__(16) uint8_t lds[kLds];
  __shared__ int lds_exp[kQueries];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, kq = lane >> 4;
  const int kv_heads = p.at.kv_heads, group = r.heads / kv_heads;
  const Partials part = partials_at<HD>(ws, r.rows, slots.all);

  Found f;
  const Class cl{group, share};
  if (!find(r, kv_heads, cl, blockIdx.x, f)) return;
  const Seq s = f.s;
  // The last tiles, which see most, first. KV heads in turn: workgroups go to the 8 XCDs in turn, so an L2
  // holds the pages of one or two heads where there are 4 or 8.
  int local = f.local;
  const int head = local % kv_heads;
  local /= kv_heads;
  const int tile = f.tiles - 1 - local % f.tiles, c = local / f.tiles;
  const int pages = tile_pages(s, group, kQueries, tile), have = chunks_of(pages, f.chunk);
  if (c == 0 && head == 0 && slots.all > 0) leave_row_parts(part, s, group, tile, kQueries, f, slots);
  if (c >= have) return;
  const int page0 = c * f.chunk, page1 = min(page0 + f.chunk, pages), steps = (page1 - page0 + PG - 1) / PG;
  const int* table = r.block_tables + (int64_t)f.seq * r.max_blocks;
  Walk walk;
  auto refill = [&](int it) {
    const int i = page0 + PG * it + lane;
    walk.set(i < page1 ? i : -1, table, r.max_blocks, p.n_pages);
  };
  if (steps > 0) refill(0);

  // The wave's queries, 16 at a time: loaded as rows, turned into operands through LDS.
  h8 qt[kN][kSteps];
#pragma unroll
  for (int k = 0; k < kN; k++) {
    if (k > 0) __syncthreads();
#pragma unroll
    for (int u0 = 0; u0 < 16 * HD / 8; u0 += 64) {
      const int u = u0 + lane, g8 = u % (HD / 8), q = u / (HD / 8);
      const int ql = wave * 16 + q, qi = tile * kQueries + ql;
      float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (qi < s.n * group)
        load8<T>(r.q, (int64_t)(s.row0 + qi / group) * r.ldq + (head * group + qi % group) * HD + g8 * 8, x);
      h8 terms[kN];
      const int e = query_terms<T, HD>(x, terms);
      if (g8 == 0) lds_exp[ql] = e;
      const int step = (g8 >> 3) * 2 + (g8 & 1), k4 = g8 >> 1 & 3;
      reinterpret_cast<h8*>(lds + wave * kQBytes)[step * 64 + k4 * 16 + q] = terms[k];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSteps; i++) qt[k][i] = reinterpret_cast<const h8*>(lds + wave * kQBytes)[i * 64 + lane];
  }
  __syncthreads();

  // (columns without a query, all zeros, go along with the last row)
  const int q0 = tile * kQueries + wave * 16, end = s.n * group, qi = q0 + n16;
  Query q;
  q.exp = lds_exp[wave * 16 + n16];
  q.lim = seen_by(s, min(qi, end - 1) / group);
  const int least = seen_by(s, min(q0, end - 1) / group);
  const int most = q0 < end ? seen_by(s, min(q0 + 15, end - 1) / group) : 0;
  const PoolAt pool(p, head);
  u4 next[kRounds];
  auto load = [&](const Page (&g)[PG]) {
#pragma unroll
    for (int i = 0; i < kRounds; i++) {
      // a page takes whole rounds, or (hd 64) half of one
      constexpr int kPer = kHead / 4096;
      const Page* from = &g[kPer > 0 ? i / (kPer > 0 ? kPer : 1) : 2 * i];
      const uint8_t* at = from->at;
      int id = from->id;
      if (kPer == 0 && tid >= 128) {
        at = g[(2 * i + 1) % PG].at;
        id = g[(2 * i + 1) % PG].id;
      }
      next[i] = *reinterpret_cast<const u4*>(at + (i * 4096 + tid * 16) % kHead);
      if (id < 0) next[i] = u4{0, 0, 0, 0};
    }
  };
  auto put = [&](int b) {
#pragma unroll
    for (int i = 0; i < kRounds; i++) reinterpret_cast<u4*>(lds + b * PG * kHead)[i * 256 + tid] = next[i];
  };
  const float scale = 1.44269504088896340736f / sqrtf((float)HD);
  f4 o[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; i++) o[i] = f4{0, 0, 0, 0};
  Page cur[PG], nxt[PG];
  auto pages_at = [&](int it, Page (&g)[PG]) {
#pragma unroll
    for (int w = 0; w < PG; w++) g[w] = pool.page(walk, PG * (it % (64 / PG)) + w);
  };
  if (steps > 0) {
    pages_at(0, cur);
    load(cur);
    put(0);
  }
  __syncthreads();
  for (int it = 0; it < steps; it++) {
    const bool more = it + 1 < steps;
    if (more) {
      if ((it + 1) % (64 / PG) == 0) refill(it + 1);
      pages_at(it + 1, nxt);
      load(nxt);
    }
    if (cur[0].index * kPage < most) {  // (the step is not behind all of the wave's queries)
      const u4* kv = reinterpret_cast<const u4*>(lds + (it & 1) * PG * kHead) + lane;
      f4 sc[PG];
#pragma unroll
      for (int w = 0; w < PG; w++) sc[w] = f4{0, 0, 0, 0};
      __builtin_amdgcn_s_setprio(1);  // (the other wave of the SIMD weighs meanwhile)
#pragma unroll
      for (int i = 0; i < kSegs; i++) {
        u4 code[PG];
#pragma unroll
        for (int w = 0; w < PG; w++) code[w] = kv[w * kHead / 16 + i * 64];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          h8 a[PG];
#pragma unroll
          for (int w = 0; w < PG; w++) a[w] = of_codes8(code[w][2 * h], code[w][2 * h + 1]);
#pragma unroll
          for (int k = 0; k < kN; k++)
#pragma unroll
            for (int w = 0; w < PG; w++)
              sc[w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[w], qt[k][2 * i + h], sc[w], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      h8 wt[PG / 2][kW];
      weigh(sc, cur, scale, whole_pages(cur, least), q, o, wt);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < kSegs; i++) {
        u4 code[PG];
#pragma unroll
        for (int w = 0; w < PG; w++) code[w] = kv[w * kHead / 16 + kHead / 32 + i * 64];
#pragma unroll
        for (int w = 0; w < PG; w += 2) {
          h8 a[4];
#pragma unroll
          for (int j = 0; j < 4; j++) a[j] = of_codes8(code[w][j], code[w + 1][j]);
          // (terms outermost: a product on the same sums as the one before it would wait for it)
#pragma unroll
          for (int k = kW - 1; k >= 0; k--)
#pragma unroll
            for (int j = 0; j < 4; j++)
              o[4 * i + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[j], wt[w / 2][k], o[4 * i + j], 0, 0, 0);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    }
    if (more) {
      put((it + 1) & 1);
#pragma unroll
      for (int w = 0; w < PG; w++) cur[w] = nxt[w];
    }
    __syncthreads();
  }

  const float l = quads_sum(q.l);
  if (qi >= end) return;
  const int row = s.row0 + qi / group, col = (head * group + qi % group) * HD;
  if (have > 1) {
    const int64_t slot = slots.first + f.slot + ((int64_t)c * kv_heads + head) * cl.tiles16(s.n) + qi / 16;
    if (slot >= slots.end) return;
    if (kq == 0) part.st[slot * 16 + n16] = f4{q.m, q.d, l, 0};
#pragma unroll
    for (int i = 0; i < kTiles; i++) *reinterpret_cast<f4*>(part.o + (slot * 16 + n16) * HD + i * 16 + kq * 4) = o[i];
  } else {
    State st;
    st.m = q.m;
    st.d = q.d;
    st.l = l;
    const State::Factor result = st.factor();
#pragma unroll
    for (int i = 0; i < kTiles; i++) store4<T>(out, row, col + i * 16 + kq * 4, result(o[i]));
  }
}

// ---- joining the chunks ---------------------------------------------------------------

// WAVES waves per (row, head): the partial sums of its chunks, each wave's in order, then the waves' in order.
// 5.5 us for 768 results (latency), 30 for 54576 (HBM).
template <int HD, int T, bool LIST, int WAVES>
__global__ __launch_bounds__(256) void merge_kernel(Rows r, Out out, List list, int kv_heads, void* ws, int slots) {
  constexpr int kLanes = HD / 4, kSub = 64 / kLanes;  // lanes with 4 dims each, and chunks that a wave takes at once
  constexpr int kParts = WAVES * kSub;
  __shared__ f4 lds_o[4][kLanes];
  __shared__ f4 lds_st[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int id = WAVES == 4 ? blockIdx.x : blockIdx.x * 4 + wave;  // (rows * heads stay below 2^26)
  const int row = id / r.heads, h = id % r.heads;
  const int first = (WAVES == 4 ? wave * kSub : 0) + lane / kLanes;  // this lane's first chunk
  if (row >= r.rows) return;
  const int group = r.heads / kv_heads, head = h / group;
  const Partials part = partials_at<HD>(ws, LIST ? 0 : r.rows, slots);
  int chunks, q;
  int64_t slot, step;
  if constexpr (LIST) {
    const int count = min(max(list.count[(int64_t)row * kv_heads + head], 0), list.top), tiles = (group + 15) / 16;
    chunks = chunks_of(count, list.chunk);
    q = h % group;
    slot = (((int64_t)row * kv_heads + head) * tiles + q / 16) * list.chunks;
    step = 1;
    if (chunks == 1 || row < r.row_start[0] || row >= r.row_start[r.nseq]) return;
  } else {
    const RowPart rp = part.rows[row];
    if (row < r.row_start[0] || row >= r.row_start[r.nseq]) return;
    Seq s;
    s.row0 = rp.row0;
    s.n = rp.n;
    s.len = rp.len;
    s.ctx = (int)min((long long)max(s.len, 0), (long long)r.max_blocks * kPage);
    q = (row - rp.row0) * group + h % group;
    const int tiles = (rp.n * group + 15) >> 4;
    if (rp.chunk < kMinChunk || rp.tile_queries < 16) return;
    chunks = chunks_of(tile_pages(s, group, rp.tile_queries, q / rp.tile_queries), rp.chunk);
    slot = rp.slot + (int64_t)head * tiles + q / 16;
    step = (int64_t)kv_heads * tiles;
    if (chunks == 1) return;
  }
  if (slot < 0 || step < 0 || slot + (chunks - 1) * step >= slots) return;  // (row starts that do not ascend)
  q &= 15;
  State j;
  auto state_of = [&](int c) { return part.st[(slot + c * step) * 16 + q]; };
  const f4 own = lane < chunks ? state_of(lane) : f4{-INFINITY, -INFINITY, 0, 0};
  j.m = own[0];
  for (int c = lane + 64; c < chunks; c += 64) j.m = fmaxf(j.m, state_of(c)[0]);
  j.m = lanes_max<64>(j.m);
  j.d = j.level(own);
  for (int c = lane + 64; c < chunks; c += 64) j.d = fmaxf(j.d, j.level(state_of(c)));
  j.d = lanes_max<64>(j.d);
  f4 x{0, 0, 0, 0};
#pragma unroll 8
  for (int c = first; c < chunks; c += kParts) {
    const f4 st = state_of(c);
    x += *reinterpret_cast<const f4*>(part.o + ((slot + c * step) * 16 + q) * HD + (lane % kLanes) * 4) * j.of_part(st);
    j.l += j.sum_of_part(st);
  }
  // lanes of the same dims, then waves
#pragma unroll
  for (int o = kLanes; o < 64; o <<= 1) {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] += __shfl_xor(x[i], o);
    j.l += __shfl_xor(j.l, o);
  }
  if constexpr (WAVES == 4) {
    if (lane < kLanes) lds_o[wave][lane] = x;
    if (lane == 0) lds_st[wave][0] = j.l;
    __syncthreads();
    if (wave > 0) return;
    if (lane < kLanes)
#pragma unroll
      for (int w = 1; w < 4; w++) x += lds_o[w][lane];
#pragma unroll
    for (int w = 1; w < 4; w++) j.l += lds_st[w][0];
  }
  if (lane < kLanes) store4<T>(out, row, (int64_t)h * HD + lane * 4, j.factor()(x));
}

// ---- launches ---------------------------------------------------------------------------

struct Grid {
  int64_t items, slots;
};

// Items and partial sums that a share may have. Tiles of all rows' queries: at most a full
// one for every `tile` and a last one for every sequence. A context of p pages makes at most p / each + 1 items of a
// tile, and 8/7 p / each if it is cut at all; all tiles' pages over `each` are share.items (but for the rounding of
// sums in f32: an eighth more).
Grid grid_of(const Layout& at, int heads, int nseq, int max_blocks, int rows, const Share& sh) {
  const int64_t group = heads / at.kv_heads, seqs = nseq < rows ? nseq : rows;
  int64_t tiles = rows * group / sh.tile + seqs;
  if (sh.most < INT_MAX) tiles = std::min(tiles, seqs * ((sh.most + sh.tile - 1) / sh.tile));
  tiles *= at.kv_heads;
  const int64_t per = (max_blocks + least_chunk(max_blocks) - 1) / least_chunk(max_blocks), cut = tiles * per,
                most = sh.items + sh.items / 8;
  return Grid{std::min(cut, tiles + most), per > 1 ? std::min(cut, 2 * most) * (sh.tile / 16) : 0};
}

// How a call is shared out: by the largest number of queries that a sequence has for a KV head. Up to 16 and up to
// kFewQueries are item_kernel's alone, one or two tiles side by side; past that it keeps the sequences of up to 16
// (16 of 2 to 32 rows, 6 queries a row: 63 us; up to 32 or 64: 67 and 66).
struct Plan {
  Share few, many;
  bool two;   // tiles side by side
  bool both;  // prompt_kernel has a share
};
Plan plan_of(int hd, int group, int64_t max_rows) {
  const int64_t most = max_rows * group;
  Plan p{};
  p.both = most > kFewQueries;
  p.two = most > 16 && !p.both;
  p.few = Share{1, p.both ? 16 : INT_MAX, p.two ? 32 : 16, few_items(hd, p.two ? 2 : 1), few_items(hd, p.two ? 2 : 1)};
  p.many = Share{17, INT_MAX, 64, many_items(hd), many_at_once(hd)};
  return p;
}

int sparse_chunk(const Layout& at, int heads, int rows, int top) {
  const int64_t all = (int64_t)rows * at.kv_heads * ((heads / at.kv_heads + 15) / 16) * top;
  const int64_t items = few_items(at.hd, 1), c = ((all + items - 1) / items + 7) & ~7ll;
  return (int)std::max(std::min(c, (int64_t)1 << 20), (int64_t)least_chunk(top));
}

template <int HD, int T>
void merge(const Rows& r, const Out& o, const List* list, int kv_heads, void* ws, int64_t slots, hipStream_t s) {
  const int64_t outs = (int64_t)r.rows * r.heads;
  const List l = list ? *list : List{};
  // Four waves a result where there are few: 768 results 24.2 against 25.5 us with one wave each, 1536 the same.
  auto go = [&](auto is_list, auto waves) {
    const unsigned blocks = (unsigned)(waves == 4 ? outs : (outs + 3) / 4);
    merge_kernel<HD, T, is_list, waves><<<blocks, 256, 0, s>>>(r, o, l, kv_heads, ws, (int)slots);
  };
  const bool wide = outs <= 1024;
  using W4 = std::integral_constant<int, 4>;
  using W1 = std::integral_constant<int, 1>;
  if (list) wide ? go(std::true_type(), W4()) : go(std::true_type(), W1());
  else wide ? go(std::false_type(), W4()) : go(std::false_type(), W1());
  PGD_HIP(hipGetLastError());
}

template <class F>
void with_types(const Pool& p, const Rows& r, F&& go) {
  auto typed = [&](auto hd) {
    if (r.type == F32) go(hd, std::integral_constant<int, F32>());
    else if (r.type == F16) go(hd, std::integral_constant<int, F16>());
    else go(hd, std::integral_constant<int, BF16>());
  };
  if (p.at.hd == 64) typed(std::integral_constant<int, 64>());
  else if (p.at.hd == 128) typed(std::integral_constant<int, 128>());
  else typed(std::integral_constant<int, 256>());
}

size_t partial_bytes(const Layout& at, int64_t slots) { return (size_t)slots * 16 * (at.hd + 4) * 4; }

}  // namespace

size_t attn_ws_bytes(const Layout& at, int heads, int nseq, int max_blocks, int rows, int max_rows) {
  // the plans of all numbers up to max_rows
  const int group = heads / at.kv_heads, most = std::min(max_rows, rows);
  int64_t slots = 0;
  for (int n : {0, std::min(kFewQueries / group, most), most}) {
    const Plan p = plan_of(at.hd, group, n);
    slots = std::max(slots, grid_of(at, heads, nseq, max_blocks, rows, p.few).slots +
                                (p.both ? grid_of(at, heads, nseq, max_blocks, rows, p.many).slots : 0));
  }
  return slots ? (size_t)rows * sizeof(RowPart) + partial_bytes(at, slots) : 0;
}

void attn(const Pool& p, const Rows& r, int max_rows, const Out& o, void* ws, hipStream_t s) {
  const Plan pl = plan_of(p.at.hd, r.heads / p.at.kv_heads, std::min(max_rows, r.rows));
  const Grid few = grid_of(p.at, r.heads, r.nseq, r.max_blocks, r.rows, pl.few);
  const Grid many = pl.both ? grid_of(p.at, r.heads, r.nseq, r.max_blocks, r.rows, pl.many) : Grid{};
  const int all = (int)(few.slots + many.slots);
  with_types(p, r, [&](auto hd, auto type) {
    constexpr int HD = decltype(hd)::value, T = decltype(type)::value;
    if (pl.both) {
      prompt_kernel<HD, T, HD == 64 ? 2 : 4><<<(unsigned)many.items, 256, 0, s>>>(p, r, o, pl.many, ws,
                                                                                 Slots{all, (int)few.slots, all});
      PGD_HIP(hipGetLastError());
    }
    const Slots own{all, 0, (int)few.slots};
    if (pl.two) item_kernel<HD, T, 2, false><<<(unsigned)few.items, 512, 0, s>>>(p, r, o, List{}, pl.few, ws, own);
    else item_kernel<HD, T, 1, false><<<(unsigned)few.items, 256, 0, s>>>(p, r, o, List{}, pl.few, ws, own);
    PGD_HIP(hipGetLastError());
    if (all > 0) merge<HD, T>(r, o, nullptr, p.at.kv_heads, ws, all, s);
  });
}

size_t attn_sparse_ws_bytes(const Layout& at, int heads, int rows, int top) {
  const int c = sparse_chunk(at, heads, rows, top), chunks = (top + c - 1) / c;
  if (chunks <= 1) return 0;
  return partial_bytes(at, (int64_t)rows * at.kv_heads * ((heads / at.kv_heads + 15) / 16) * chunks);
}

// Lists are cut only while there are fewer of them than items, then into at most top / c + 1 chunks of c pages, whose
// top / c is at most items over lists; and no chunk is shorter than the least.
size_t attn_sparse_ws_most(const Layout& at, int heads, int rows, int top) {
  if (top <= kOneChunk) return 0;
  const int64_t items = few_items(at.hd, 1), lists = (int64_t)rows * at.kv_heads * ((heads / at.kv_heads + 15) / 16),
                cut = std::min(lists, items - 1), per = (top + least_chunk(top) - 1) / least_chunk(top);
  return partial_bytes(at, std::min(cut * per, items + cut));
}

void attn_sparse(const Pool& p, const Rows& r, int top, const int* sel, const int* count, const Out& o, void* ws,
                 hipStream_t s) {
  const int c = sparse_chunk(p.at, r.heads, r.rows, top), chunks = (top + c - 1) / c;
  const int64_t items = (int64_t)r.rows * p.at.kv_heads * ((r.heads / p.at.kv_heads + 15) / 16) * chunks;
  const List list{sel, count, top, c, chunks};
  with_types(p, r, [&](auto hd, auto type) {
    constexpr int HD = decltype(hd)::value, T = decltype(type)::value;
    item_kernel<HD, T, 1, true><<<(unsigned)items, 256, 0, s>>>(p, r, o, list, Share{}, ws, Slots{(int)items, 0, (int)items});
    PGD_HIP(hipGetLastError());
    if (chunks > 1) merge<HD, T>(r, o, &list, p.at.kv_heads, ws, items, s);
  });
}

}  // namespace kv8
}  // namespace pgd
