// Paged key-value cache: appending new tokens with their position rotation,
// and attention of one new token per row over the cache.
//
// Cache layout: k and v are (num_pages, kv_heads, page_size, head_dim), so the
// tokens of one head in one page are one contiguous run; a row's tokens are
// found through its page table, position p at slot p % page_size of page
// table[p / page_size].
#pragma once

#include <type_traits>

#include "common.cuh"
#include "sgmv_grid.cuh"
#include "sgmv_stream.cuh"

namespace plora {

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, 1994).
struct FastDiv {
  uint32_t d, m, s;
  __host__ void set(uint32_t div) {
    d = div;
    s = 0;
    while ((1ull << s) < div) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - div)) / div + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

struct PagedView {
  void *k, *v;
  const int32_t* table;   // (rows, max_pages)
  int64_t table_stride;   // entries between rows
  int64_t k_page, v_page; // elements between pages
  int64_t capacity;       // positions a row's table reaches: max_pages * page_size
  int32_t num_pages, kv_heads, page_size, dim;
  FastDiv page;
};

// Elements of one 16-byte chunk as floats.
template <typename T>
struct Chunk;
template <>
struct Chunk<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const uint4& u, float* f) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 store(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float f) { return f; }
};
template <>
struct Chunk<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ uint4 store(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float f) { return __float2bfloat16_rn(f); }
};
template <>
struct Chunk<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const uint4& u, float* f) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 store(const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float f) { return __float2half_rn(f); }
};

// ---------------------------------------------------------------- append
// Token (b, m), m < new_lens[b], has position past_lens[b] + m.  Its queries
// and keys are rotated by the angle position * f_i of each pair i of head
// elements, (x, y) -> (x cos - y sin, y cos + x sin), keys and values go to the
// row's pages, rotated queries (and keys, if wanted) to dense outputs.
//
// The angle is kept as a fraction of a turn: phases[i] = round(f_i / 2 pi * 2^64),
// and position * phases[i] mod 2^64 is an exact integer product, so far
// positions lose nothing (a 32-bit float product is off by 2^-24 of the angle,
// 0.008 rad at position 131072).
constexpr int kAppendThreads = 256;
constexpr int kAppendTokens = 4;   // most tokens of a CTA
constexpr int kAppendPairs = 128;  // most rotated pairs of a head (head_dim <= 256)

struct AppendParams {
  PagedView c;
  const void *q, *k, *v;
  void *q_out, *k_out;  // dense (rows, max_new, heads, dim); q_out null when q is, k_out may be null
  int64_t q_row, q_tok, q_head, k_row, k_tok, k_head, v_row, v_tok, v_head;  // strides in elements
  const int32_t *past, *news;  // news null: every row has max_new tokens
  const uint64_t* phases;      // null: no rotation (pairs 0)
  int32_t q_heads, pairs, interleaved, max_new, tokens, cta_tokens;
  float scale;
  FastDiv by_new, by_item, by_head;  // max_new; items of a token; items of a head
};

// Rotates element j of a head vector from its parts (the slow path: pairs that
// do not fill 16-byte chunks).
template <typename T>
__device__ __forceinline__ float rotated_at(const T* x, int j, const float2* cs, int pairs, int interleaved) {
  const float a = Chunk<T>::get(x[j]);
  if (j >= 2 * pairs) return a;
  const int i = interleaved ? j >> 1 : (j < pairs ? j : j - pairs);
  const bool first = interleaved ? !(j & 1) : j < pairs;
  const float b = Chunk<T>::get(x[interleaved ? j ^ 1 : (first ? j + pairs : j - pairs)]);
  return first ? a * cs[i].x - b * cs[i].y : a * cs[i].x + b * cs[i].y;
}

// One CTA takes cta_tokens tokens; a thread's item is two 16-byte chunks of a
// head vector, which hold whole pairs when VEC (each element is then read
// once): chunks c and c + pairs / N in halves, 2c and 2c + 1 interleaved.  The
// cosines of a token are computed once and shared by all of its heads: for each
// head anew they would take longer than the bytes.  Bound by HBM for prompts (64 of
// up to 1024 tokens, 48 heads of 128, bf16, 1.48 GB: 242 us, 6.1 TB/s), by three
// dependent loads for single tokens (256 of them 3.5 us).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kAppendThreads) paged_append_kernel(const AppendParams p) {
  constexpr int N = Chunk<T>::N;
  __shared__ float2 cs[kAppendTokens][kAppendPairs];
  __shared__ int32_t s_page[kAppendTokens];  // -2: padding; -1: no place in the cache
  __shared__ int32_t s_slot[kAppendTokens];
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * p.cta_tokens;
  const int nt = min(p.cta_tokens, p.tokens - t0);
  const int pairs = p.pairs, dim = p.c.dim;

  for (int i = tid; i < nt * max(pairs, 1); i += kAppendThreads) {
    const int tok = pairs ? i / pairs : i, pr = pairs ? i - tok * pairs : 0;
    const int b = p.by_new.div(t0 + tok), m = t0 + tok - b * p.max_new;
    const int64_t pos = (int64_t)p.past[b] + m;
    if (pairs) {
      const uint64_t turn = (uint64_t)pos * p.phases[pr];
      float s, c;
      sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);  // half turns in [-1, 1]
      cs[tok][pr] = make_float2(c * p.scale, s * p.scale);
    }
    if (pr == 0) {
      int page = -2, slot = 0;
      if (m < (p.news ? min(p.news[b], p.max_new) : p.max_new)) {
        page = -1;
        if (pos >= 0 && pos < p.c.capacity) {
          const uint32_t e = p.c.page.div((uint32_t)pos);
          slot = (int)((uint32_t)pos - e * p.c.page.d);
          page = p.c.table[b * p.c.table_stride + e];
          if ((uint32_t)page >= (uint32_t)p.c.num_pages) page = -1;
        }
        if (page < 0) raise_status(PLORA_DEV_PAGE_RANGE);
      }
      s_page[tok] = page;
      s_slot[tok] = slot;
    }
  }
  __syncthreads();

  const int per_token = (int)p.by_item.d, per_head = (int)p.by_head.d;
  const int rot = VEC && !p.interleaved ? pairs / N : 0;  // items of a head that hold both halves of their pairs
  for (int i = tid; i < nt * per_token; i += kAppendThreads) {
    const int tok = p.by_item.div(i);
    int r = i - tok * per_token;
    int head = p.by_head.div(r);
    const int c = r - head * per_head;
    const int t = t0 + tok, b = p.by_new.div(t), m = t - b * p.max_new;
    const int page = s_page[tok];
    // which tensor: q heads, then k heads, then v heads
    const T* x;
    T *dense = nullptr, *cache = nullptr;
    bool turn = pairs > 0;
    if (head < p.q_heads) {
      x = (const T*)p.q + b * p.q_row + m * p.q_tok + head * p.q_head;
      dense = (T*)p.q_out + ((int64_t)t * p.q_heads + head) * dim;
    } else {
      head -= p.q_heads;
      const bool key = head < p.c.kv_heads;
      if (!key) head -= p.c.kv_heads;
      const int64_t at = ((int64_t)head * p.c.page_size + s_slot[tok]) * dim;
      if (key) {
        x = (const T*)p.k + b * p.k_row + m * p.k_tok + head * p.k_head;
        if (p.k_out) dense = (T*)p.k_out + ((int64_t)t * p.c.kv_heads + head) * dim;
        if (page >= 0) cache = (T*)p.c.k + page * p.c.k_page + at;
      } else {
        x = (const T*)p.v + b * p.v_row + m * p.v_tok + head * p.v_head;
        if (page >= 0) cache = (T*)p.c.v + page * p.c.v_page + at;
        turn = false;
      }
    }
    const int first = c < rot ? c * N : 2 * c * N, e1 = first + (c < rot ? pairs : N);
    const bool two = e1 < dim;
    uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
    if (page != -2) {
      if (VEC || !turn) {
        u0 = *reinterpret_cast<const uint4*>(x + first);
        if (two) u1 = *reinterpret_cast<const uint4*>(x + e1);
        if (turn) {
          float a[N], d[N], y0[N], y1[N];
          Chunk<T>::load(u0, a);
          Chunk<T>::load(u1, d);
          if (p.interleaved) {
#pragma unroll
            for (int j = 0; j < N; j += 2) {
              const float2 w = first < 2 * pairs ? cs[tok][(first + j) >> 1] : make_float2(1.f, 0.f);
              const float2 z = e1 < 2 * pairs ? cs[tok][(e1 + j) >> 1] : make_float2(1.f, 0.f);
              y0[j] = a[j] * w.x - a[j + 1] * w.y, y0[j + 1] = a[j + 1] * w.x + a[j] * w.y;
              y1[j] = d[j] * z.x - d[j + 1] * z.y, y1[j + 1] = d[j + 1] * z.x + d[j] * z.y;
            }
            if (first < 2 * pairs) u0 = Chunk<T>::store(y0);
            if (e1 < 2 * pairs) u1 = Chunk<T>::store(y1);
          } else if (c < rot) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
              const float2 w = cs[tok][first + j];
              y0[j] = a[j] * w.x - d[j] * w.y;
              y1[j] = d[j] * w.x + a[j] * w.y;
            }
            u0 = Chunk<T>::store(y0);
            u1 = Chunk<T>::store(y1);
          }
        }
      } else {
        float y[N];
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = rotated_at(x, first + j, cs[tok], pairs, p.interleaved);
        u0 = Chunk<T>::store(y);
        if (two) {
#pragma unroll
          for (int j = 0; j < N; ++j) y[j] = rotated_at(x, e1 + j, cs[tok], pairs, p.interleaved);
          u1 = Chunk<T>::store(y);
        }
      }
    }
    if (dense) {
      *reinterpret_cast<uint4*>(dense + first) = u0;
      if (two) *reinterpret_cast<uint4*>(dense + e1) = u1;
    }
    if (cache) {
      *reinterpret_cast<uint4*>(cache + first) = u0;
      if (two) *reinterpret_cast<uint4*>(cache + e1) = u1;
    }
  }
}

// ---------------------------------------------------------------- attention
// out[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j over the last
// min(window, seq_lens[b]) of a row's seq_lens[b] cached tokens; zeros where
// there are none.  One pass over the cache with a running maximum and sum.
//
// Bound by HBM: the cache is read once, 4 * group flops for each 2 * elem
// bytes.  The rows' lengths are known on the device only, so the work is cut
// there.  An item is a row and a key-value head (or a block of its query
// heads), a tile 16 of its tokens; every item has at least one (empty) tile, so
// rows without tokens are written too.  The list of all items' tiles is cut into
// segments, which warps stream through a ring of shared-memory stages of their
// own, with no barrier between them.
//
// Where there is much to do, the first 13/16 of the list are dealt in
// equal segments to the grid's warps and the rest in small ones to whoever asks
// next: SMs of a GPC share its way to memory, and with equal shares alone the
// slowest warp of a 2 GB call ended 17 % after the mean (325 and 277 us).  The
// segments' bounds depend on the lengths only, not on who takes them, and an item
// cut by them is put together in the order of the list (attn_join_kernel), so
// results do not depend on timing.
//
// Few items of few tiles, which the SMs hold at once, need no list: a cluster of
// CTAs takes an item, its warps equal parts of the tiles, and puts them together
// through distributed shared memory, in one launch.
constexpr int kAttnTile = 16;

// 2^x to 2 ulp; results below 2^-126 are zero, next to a largest term of 1.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct AttnParams {
  PagedView c;
  const void* q;
  void* out;  // dense (rows, heads, dim)
  const int32_t* seq_lens;
  int64_t q_row, q_head;
  int32_t rows, group, blocks, block_heads, window;  // blocks of block_heads query heads cover a group
  float scale_log2;                                  // scale * log2(e)
  int32_t direct;                                    // CTAs of an item's cluster; 0: by the list
  // workspace
  struct AttnWork* work;
  int64_t* before;  // (rows): tiles of the rows before, per item
  int4* cut;        // items cut by segments: row, item of the row, segment it begins in, segments; those of
  int cut_room;     // more than kJoinAlone segments from the end of the list (of cut_room entries) backwards
  // a segment's parts of cut items (0: begun in an earlier one, 1: begun here): the
  // sums of block_heads heads, and for each its maximum (in units of scale_log2)
  // and sum of probabilities
  float* part_o;    // (segments, 2, block_heads, dim)
  float2* part_ml;  // (segments, 2, block_heads)
};

// The list of tiles and its segments: `dealt` of base or (the first rem) base + 1
// tiles, then `asked` of `chunk` tiles (the last one of what is left).
struct AttnWork {
  int64_t total;
  int dealt, base, rem, asked, chunk;
  int next;  // the next segment to be asked for
  int cuts[2];  // entries of the list of cut items, from its begin and from its end
};

struct AttnRow {
  int lo, n;   // tokens [lo, n)
  int t0, t1;  // tiles [t0, t1), at least one
};
__device__ __forceinline__ AttnRow attn_row(const AttnParams& p, int64_t n) {  // n: its seq_lens
  AttnRow r;
  n = n < 0 ? 0 : (n > p.c.capacity ? p.c.capacity : n);
  r.n = (int)n;
  r.lo = p.window > 0 ? max(0, r.n - p.window) : 0;
  r.t0 = r.lo / kAttnTile;
  r.t1 = max(r.t0 + 1, (r.n + kAttnTile - 1) / kAttnTile);
  return r;
}

// A position in the list of all tiles: rows, their key-value heads, blocks of
// a group's query heads, tiles.
struct AttnCursor {
  int row, kv, blk, tile;
  int next_n;  // the next row's length, on its way since this row began
  AttnRow r;
  __device__ __forceinline__ void enter(const AttnParams& p, int64_t n) {
    r = attn_row(p, n);
    next_n = row + 1 < p.rows ? p.seq_lens[row + 1] : 0;
  }
  __device__ __forceinline__ void next(const AttnParams& p) {
    if (++tile < r.t1) return;
    if (++blk == p.blocks) {
      blk = 0;
      if (++kv == p.c.kv_heads) {
        kv = 0;
        if (++row < p.rows) enter(p, next_n);
      }
    }
    tile = r.t0;
  }
};

// Sum over the CTA's threads before this one (exclusive) and over all of them.
template <int WARPS, typename V>
__device__ __forceinline__ V block_scan(V v, V* s_warp, V* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += u;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  V before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += s_warp[w];
    sum += s_warp[w];
  }
  *total = sum;
  return before + incl - v;
}

// Segments that a call may have, for `warps` of the grid and block_heads heads: a
// part costs 4 * block_heads * dim bytes and a tile 64 * dim, so small segments are
// as many as keep the parts below a sixteenth of the cache's bytes.
__host__ __device__ constexpr int attn_asked_max(int warps, int block_heads) {
  return warps * (block_heads <= 4 ? 4 : (block_heads <= 8 ? 2 : 1));
}
constexpr int kAttnPlanThreads = 1024;
constexpr int kAttnDealOnly = 32;   // tiles a warp up to which all are dealt
constexpr int kAttnChunk = 8;       // smallest chunk: a loader's lead of up to 5 tiles then spans two segments
constexpr int kAttnDirect = 8;      // most tiles of a warp without a list
constexpr int kAttnAsk = 4;         // tiles ahead of which the next segment is asked for
static_assert(kAttnChunk > kAttnAsk && kAttnDealOnly > 2 * kAttnAsk, "segments that are followed by others are longer");

// Counts the tiles of the rows and cuts their list.  One CTA; 4 us, mostly launch
// and one load.
__global__ void __launch_bounds__(kAttnPlanThreads) attn_plan_kernel(const AttnParams p, int warps) {
  __shared__ int64_t s_warp[kAttnPlanThreads / 32];
  griddep_wait();
  griddep_launch();
  int64_t tiles = 0;
  for (int first = 0; first < p.rows; first += kAttnPlanThreads) {
    const int row = first + threadIdx.x;
    int64_t n = 0, sum;
    if (row < p.rows) {
      const AttnRow r = attn_row(p, p.seq_lens[row]);
      n = r.t1 - r.t0;
    }
    const int64_t before = block_scan<kAttnPlanThreads / 32>(n, s_warp, &sum);
    if (row < p.rows) p.before[row] = tiles + before;
    tiles += sum;
  }
  if (threadIdx.x == 0) {
    AttnWork w;
    w.total = tiles * p.c.kv_heads * p.blocks;
    w.next = w.cuts[0] = w.cuts[1] = 0;
    if (w.total < (int64_t)warps * kAttnDealOnly) {
      w.dealt = (int)(w.total < warps ? w.total : warps);
      w.base = (int)w.total / w.dealt;  // total < 32 warps here
      w.rem = (int)w.total - w.base * w.dealt;
      w.asked = 0, w.chunk = 1;
    } else {
      w.dealt = warps;
      w.base = (int)(w.total / 16 * 13 / warps);
      w.rem = 0;
      const int64_t rest = w.total - (int64_t)w.base * warps;
      const int most = attn_asked_max(warps, p.block_heads);
      const int64_t chunk = (rest + most - 1) / most;
      w.chunk = (int)max(chunk, (int64_t)max(kAttnChunk, p.block_heads));
      w.asked = (int)((rest + w.chunk - 1) / w.chunk);
    }
    *p.work = w;
  }
}

// A segment of the list: tiles [begin, begin + count) from `at` on.
struct AttnSegment {
  AttnCursor at;
  int id, count;
  int64_t begin;
};

// What a warp knows of the list.
struct AttnList {
  AttnWork w;
  __device__ __forceinline__ void read(const AttnParams& p) {
    w.total = ld_cg_i64(&p.work->total);
    w.dealt = ld_cg_i32(&p.work->dealt), w.base = ld_cg_i32(&p.work->base), w.rem = ld_cg_i32(&p.work->rem);
    w.asked = ld_cg_i32(&p.work->asked), w.chunk = ld_cg_i32(&p.work->chunk);
  }
  __device__ __forceinline__ int64_t dealt_tiles() const { return (int64_t)w.dealt * w.base + w.rem; }
  // The segment that holds tile x.
  __device__ __forceinline__ int holder(int64_t x) const {
    if (x >= dealt_tiles()) return w.dealt + (int)((x - dealt_tiles()) / w.chunk);
    const int64_t split = (int64_t)w.rem * (w.base + 1);
    return x < split ? (int)(x / (w.base + 1)) : w.rem + (int)((x - split) / w.base);
  }
  // Segment id < dealt + asked.  Warp-collective.
  __device__ __forceinline__ AttnSegment segment(const AttnParams& p, int id) const {
    AttnSegment s;
    s.id = id;
    if (id < w.dealt) {
      s.begin = (int64_t)id * w.base + min(id, w.rem);
      s.count = w.base + (id < w.rem ? 1 : 0);
    } else {
      s.begin = dealt_tiles() + (int64_t)(id - w.dealt) * w.chunk;
      s.count = (int)min((int64_t)w.chunk, w.total - s.begin);
    }
    // the last row that begins at or before s.begin: 32 probes a round
    const int lane = threadIdx.x & 31, per_row = p.c.kv_heads * p.blocks;
    int lo = 0, hi = p.rows;
    int64_t first = 0;  // tiles before row lo
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
      int64_t v = 0;
      bool le = false;
      if (at < hi) {
        v = ld_cg_i64(p.before + at) * per_row;
        le = v <= s.begin;
      }
      const int k = __popc(__ballot_sync(0xffffffffu, le));
      if (k) first = __shfl_sync(0xffffffffu, v, k - 1);
      lo += k * step;
      hi = min(hi, lo + step);
    }
    s.at.row = lo;
    s.at.enter(p, p.seq_lens[lo]);
    const int n = s.at.r.t1 - s.at.r.t0;
    const int rest = (int)(s.begin - first), item = rest / n;
    s.at.kv = item / p.blocks;
    s.at.blk = item - s.at.kv * p.blocks;
    s.at.tile = s.at.r.t0 + rest - item * n;
    return s;
  }
};

// A warp's walk through its segments: the one that it computes, and the next,
// into which its loader may have run ahead.
struct AttnWalk {
  AttnList list;
  AttnSegment cur, nxt;
  int asked;      // lane 0: the segment asked for last
  bool more;      // there may be another one
  bool have_nxt;
  // False when this warp has nothing to do.
  __device__ __forceinline__ bool start(const AttnParams& p) {
    more = have_nxt = false;
    if (p.direct) {
      const int item = blockIdx.x / p.direct, rank = blockIdx.x - item * p.direct, per_row = p.c.kv_heads * p.blocks;
      const int parts = p.direct * (blockDim.x >> 5), id = (threadIdx.x >> 5) * p.direct + rank;
      cur.at.row = item / per_row;
      cur.at.kv = (item - cur.at.row * per_row) / p.blocks;
      cur.at.blk = item - cur.at.row * per_row - cur.at.kv * p.blocks;
      cur.at.enter(p, p.seq_lens[cur.at.row]);
      const int n = cur.at.r.t1 - cur.at.r.t0, first = (int)((int64_t)n * id / parts);
      cur.at.tile = cur.at.r.t0 + first;
      cur.id = 0, cur.begin = 0;
      cur.count = (int)((int64_t)n * (id + 1) / parts) - first;
      return cur.count > 0;
    }
    list.read(p);
    // few segments spread over the SMs
    const int id = (threadIdx.x >> 5) * gridDim.x + blockIdx.x;
    if (id >= list.w.dealt) return false;
    more = list.w.asked > 0;
    cur = list.segment(p, id);
    return true;
  }
  // Called before each copy of a loader with `left` tiles to start: asks for the
  // next segment a few tiles ahead (every one but the last is longer, and nothing is
  // asked for in that one), and with nothing left moves the loader to it.
  __device__ __forceinline__ bool look_ahead(const AttnParams& p, int left) {
    if (!more) return false;
    if (left == kAttnAsk) ask(p);
    if (left > 0) return false;
    const int id = __shfl_sync(0xffffffffu, asked, 0), ids = list.w.dealt + list.w.asked;
    more = id + 1 < ids;
    if (id >= ids) return false;
    nxt = list.segment(p, id);
    have_nxt = true;
    return true;
  }
  __device__ __forceinline__ void ask(const AttnParams& p) {
    if ((threadIdx.x & 31) == 0) asked = list.w.dealt + atomicAdd(&p.work->next, 1);
  }
  __device__ __forceinline__ bool step() {
    if (!have_nxt) return false;
    cur = nxt, have_nxt = false;
    return true;
  }
};

// Two fused products at once.
__device__ __forceinline__ float2 fma2(const float2& a, const float2& b, const float2& c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// cp_async16 that writes zeros instead where `ok` is false.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared-memory layout of a tile: blocks of 128 bytes of its 16 rows, block by
// block; within a block the 16-byte chunks of a row are exchanged by row & 7 (the
// TMA's 128-byte swizzle), so that 8 rows of one chunk lie in 8 bank groups.
template <int EB, int DP>
struct AttnTileCfg {
  static constexpr int kChunks = DP * EB / 16;  // of a padded row
  static constexpr int kTileBytes = kAttnTile * DP * EB;
  static constexpr int kStageBytes = 2 * kTileBytes;  // keys, values
  static __device__ __forceinline__ uint32_t offset(int row, int chunk) {
    return (chunk >> 3) * (kAttnTile * 128) + row * 128 + (((chunk ^ row) & 7) << 4);
  }
};

// Copies the tiles of a share into a warp's stages, any page size and head
// size: 16 bytes a lane (cp.async).  The page of a tile's tokens is looked up one
// tile ahead (lane l: token l & 15).
template <int EB, int DP>
struct AttnCopyLoader {
  using Tile = AttnTileCfg<EB, DP>;
  AttnCursor at;
  int left;
  // of this lane's token of tile `at`: page (-1: reads as zeros), byte offsets of its
  // heads in the two caches
  int page;
  int64_t k_at, v_at;

  __device__ __forceinline__ void start(const AttnParams& p, const AttnSegment& s) {
    at = s.at, left = s.count;
    look_up(p);
  }
  __device__ __forceinline__ void look_up(const AttnParams& p) {
    page = -1, k_at = v_at = 0;
    if (left <= 0) return;
    const int pos = at.tile * kAttnTile + (threadIdx.x & 15);
    if (pos >= at.r.lo && pos < at.r.n) {
      const int e = p.c.page.div(pos);
      page = p.c.table[at.row * p.c.table_stride + e];
      if ((uint32_t)page >= (uint32_t)p.c.num_pages) {
        raise_status(PLORA_DEV_PAGE_RANGE);
        page = -1;
      } else {
        const int inner = (at.kv * p.c.page_size + pos - e * p.c.page_size) * p.c.dim;
        k_at = (page * p.c.k_page + inner) * EB;
        v_at = (page * p.c.v_page + inner) * EB;
      }
    }
  }
  // Starts the copies of tile `at` (none past the share's end) and steps on.
  __device__ __forceinline__ void issue(const AttnParams& p, uint32_t stage) {
    if (left > 0) {
      constexpr int LANES = Tile::kChunks < 32 ? Tile::kChunks : 32;  // lanes of a row
      const int lane = threadIdx.x & 31, lc = lane % LANES;
      const bool live = page >= 0;
#pragma unroll
      for (int r0 = 0; r0 < kAttnTile; r0 += 32 / LANES) {
        const int row = r0 + lane / LANES;
        const bool ok = __shfl_sync(0xffffffffu, live, row);
        const char* k = (const char*)p.c.k + __shfl_sync(0xffffffffu, k_at, row);
        const char* v = (const char*)p.c.v + __shfl_sync(0xffffffffu, v_at, row);
#pragma unroll
        for (int c = lc; c < Tile::kChunks; c += LANES) {
          if (c * (16 / EB) < p.c.dim) {  // columns past dim stay zero
            const uint32_t d = stage + Tile::offset(row, c);
            cp_async16_or_zero(d, k + c * 16, ok);
            cp_async16_or_zero(d + Tile::kTileBytes, v + c * 16, ok);
          }
        }
      }
      at.next(p);
      --left;
      look_up(p);
    }
    cp_async_commit();
  }
};

// The same by TMA, for pages of whole tiles and heads of DP elements: one lane
// starts two copies a tile, where the copies above cost the warp ~250
// instructions.  The maps view the cache as (64 elements, slot, 64-element block,
// kv head, page); a page outside the cache is an out-of-range coordinate, which
// reads as zeros.
template <int DP>
struct AttnTmaLoader {
  using Tile = AttnTileCfg<2, DP>;
  AttnCursor at;
  int left;
  int page, slot;  // of tile `at`

  __device__ __forceinline__ void start(const AttnParams& p, const AttnSegment& s) {
    at = s.at, left = s.count;
    look_up(p);
  }
  __device__ __forceinline__ void look_up(const AttnParams& p) {
    if (left <= 0) return;
    page = p.c.num_pages, slot = 0;
    const int pos = at.tile * kAttnTile;
    if (pos < at.r.n) {
      const int e = p.c.page.div(pos);
      slot = pos - e * p.c.page_size;
      page = p.c.table[at.row * p.c.table_stride + e];
      if ((uint32_t)page >= (uint32_t)p.c.num_pages) {
        raise_status(PLORA_DEV_PAGE_RANGE);
        page = p.c.num_pages;
      }
    }
  }
  // Lane 0 starts the copies of tile `at`, completing on `bar`; all step on.
  __device__ __forceinline__ void issue(const AttnParams& p, const CUtensorMap* mk, const CUtensorMap* mv,
                                        uint32_t stage, uint64_t* bar) {
    if (left <= 0) return;
    if ((threadIdx.x & 31) == 0) {
      mbar_arrive_expect_tx(bar, Tile::kStageBytes);
      tma_load_tile(stage, mk, bar, slot, at.kv, page);
      tma_load_tile(stage + Tile::kTileBytes, mv, bar, slot, at.kv, page);
    }
    at.next(p);
    --left;
    look_up(p);
  }
  static __device__ __forceinline__ void tma_load_tile(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int slot,
                                                       int kv, int page) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %3, %5, %6}], [%2];" ::"r"(dst),
        "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(slot), "r"(kv), "r"(page)
        : "memory");
  }
};

constexpr int kJoinAlone = 32;  // parts that one warp joins

// Where the sums of an item go whose part of segment `s` ends with its i-th tile.
struct AttnPlace {
  bool whole;   // to the output
  float* sums;  // else here, rows of `pitch`
  float2* ml;
  int pitch;
};
// Direct: the warp's ring (rows of DP + 4 floats: fragment rows then fall into
// different banks) and its row of `s_ml`.
template <int DP>
__device__ __forceinline__ AttnPlace attn_place(const AttnParams& p, const AttnList& list, const AttnSegment& s,
                                                const AttnCursor& at, int i, bool begun, bool done, float* ring,
                                                float2* s_ml) {
  AttnPlace o;
  if (p.direct) {
    __syncwarp();  // the last tile has been read
    o.whole = false, o.sums = ring, o.ml = s_ml, o.pitch = DP + 4;
    return o;
  }
  o.whole = begun && done;
  const int64_t part = (s.id * 2ll + (begun ? 1 : 0)) * p.block_heads;
  o.sums = p.part_o + part * p.c.dim, o.ml = p.part_ml + part, o.pitch = p.c.dim;
  if (begun && !done && (threadIdx.x & 31) == 0) {  // it goes on in the next segments, to the one of its last tile
    const int segments = list.holder(s.begin + i + (at.r.t1 - 1 - at.tile)) - s.id + 1;
    const int far = segments > kJoinAlone, n = atomicAdd(&p.work->cuts[far], 1);
    p.cut[far ? p.cut_room - 1 - n : n] = make_int4(at.row, at.kv * p.blocks + at.blk, s.id, segments);
  }
  return o;
}

// Direct: the cluster's warps' sums of its item, added in the order of CTAs and
// warps.  Every CTA works out the parts' weights for itself, and takes a share of the
// elements, four of a head a thread.  `rings`: of this CTA, `pitch` bytes apart;
// s_ml[warp][head].
constexpr int kAttnClusterCtas = 8;
template <typename T, int WARPS, int HEADS, int DP>
__device__ __forceinline__ void attn_gather(const AttnParams& p, const unsigned char* rings, int pitch,
                                            const float2 (*s_ml)[HEADS]) {
  __shared__ float s_f[kAttnClusterCtas * WARPS][HEADS];  // of a part: weight / sum of all
  cluster_sync();
  const int item = blockIdx.x / p.direct, rank = blockIdx.x - item * p.direct, per_row = p.c.kv_heads * p.blocks;
  const int row = item / per_row, kv = (item - row * per_row) / p.blocks, blk = item - row * per_row - kv * p.blocks;
  const int h0 = blk * p.block_heads, nh = min(p.block_heads, p.group - h0), quads = p.c.dim / 4;
  const int parts = p.direct * WARPS, lane = threadIdx.x & 31;
  for (int h = threadIdx.x >> 5; h < nh; h += WARPS) {
    constexpr int PER = (kAttnClusterCtas * WARPS + 31) / 32;
    float2 ml[PER];
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = lane + 32 * k;
      ml[k] = make_float2(-INFINITY, 0.f);
      if (i < parts) ml[k] = ld_cluster_f2(cluster_map(smem_u32(&s_ml[i % WARPS][h]), i / WARPS));
      top = fmaxf(top, ml[k].x);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      ml[k].x = exp2_fast(ml[k].x - base);
      sum += ml[k].y * ml[k].x;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // NaN stays
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (lane + 32 * k < parts) s_f[lane + 32 * k][h] = ml[k].x * inv;
  }
  __syncthreads();
  for (int t = rank * WARPS * 32 + threadIdx.x; t < nh * quads; t += p.direct * WARPS * 32) {
    const int h = t / quads, e = (t - h * quads) * 4;
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t own = smem_u32(rings) + (h * (DP + 4) + e) * 4;
    for (int c = 0; c < p.direct; ++c) {
      const uint32_t from = cluster_map(own, c);
      constexpr int AT_ONCE = WARPS < 8 ? WARPS : 8;
      static_assert(WARPS % AT_ONCE == 0, "");
#pragma unroll 1
      for (int w0 = 0; w0 < WARPS; w0 += AT_ONCE) {
        float4 v[AT_ONCE];
#pragma unroll
        for (int w = 0; w < AT_ONCE; ++w) v[w] = ld_cluster_f4(from + (w0 + w) * pitch);
#pragma unroll
        for (int w = 0; w < AT_ONCE; ++w) {
          const float f = s_f[c * WARPS + w0 + w][h];
          if (f == 0.f) continue;  // a warp without tiles, whose ring holds no sums
          o[0] += v[w].x * f, o[1] += v[w].y * f, o[2] += v[w].z * f, o[3] += v[w].w * f;
        }
      }
    }
    T* out = (T*)p.out + (((int64_t)row * p.c.kv_heads + kv) * p.group + h0 + h) * p.c.dim + e;
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = Chunk<T>::put(o[k]);
  }
  cluster_sync();  // no CTA leaves while another reads it
}

template <int DP, int H>
struct AttnSimtCfg {
  using Tile = AttnTileCfg<4, DP>;
  static constexpr int kHeads = H;  // query heads of a block
  static constexpr int kStages = DP == 64 ? 3 : 2;
  static constexpr int kWarps = DP == 256 ? 3 : (DP == 128 ? 6 : 8);
  static constexpr int kQBytes = kHeads * DP * 4, kPBytes = kAttnTile * kHeads * 8;
  static constexpr int kWarpBytes = kStages * Tile::kStageBytes + kQBytes + kPBytes;
  static constexpr int kSmemBytes = kWarps * kWarpBytes;
};

// CUDA-core attention for fp32 (TF32 products would lose 13 bits of it).
// Scores: lanes l and l + 16 take token l & 15, each half of the head's
// elements.  Sums: a lane owns DP / 32 elements of all heads.  Products come in
// pairs (fma.rn.f32x2): issue slots are the bound, not memory (1.06 GB, groups of
// three heads of 128: 197 us, 5.4 TB/s; 340 us by single products).
template <int DP, int H>
__global__ void __launch_bounds__(AttnSimtCfg<DP, H>::kWarps * 32, 1) attn_simt_kernel(const AttnParams p) {
  using T = float;
  using Cfg = AttnSimtCfg<DP, H>;
  using Tile = AttnTileCfg<4, DP>;
  constexpr int N = 4, E = DP / 32, W = E < 4 ? E : 4;  // elements of a lane, W in a run
  extern __shared__ __align__(128) unsigned char attn_smem[];
  __shared__ float2 s_ml[Cfg::kWarps][H];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* mine = attn_smem + warp * Cfg::kWarpBytes;
  float* sq = reinterpret_cast<float*>(mine + Cfg::kStages * Tile::kStageBytes);  // [H][DP]
  float2* sp = reinterpret_cast<float2*>(sq + H * DP);                            // [16][H]: twice the same
  if (p.c.dim < DP)  // columns that no copy fills
    for (int i = lane; i < Cfg::kWarpBytes / 16; i += 32) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
  if (lane < H) s_ml[warp][lane] = make_float2(-INFINITY, 0.f);
  __syncwarp();
  griddep_wait();
  griddep_launch();
  AttnWalk walk;
  const bool busy = walk.start(p);
  if (!busy && !p.direct) return;
  auto load_q = [&](const AttnCursor& c) {
    const int first = c.blk * p.block_heads, n = min(p.block_heads, p.group - first), quads = p.c.dim / 4;
    const float* q = (const float*)p.q + c.row * p.q_row + (c.kv * p.group + first) * p.q_head;
    for (int j = lane; j < H * (DP / 4); j += 32) {
      const int h = j / (DP / 4), e = j % (DP / 4);
      const bool ok = h < n && e < quads;
      cp_async16_or_zero(smem_u32(sq + h * DP + e * 4), ok ? q + h * p.q_head + e * 4 : q, ok);
    }
    cp_async_commit();
  };
  if (busy) load_q(walk.cur.at);  // on their way while the first pages are looked up
  AttnCopyLoader<4, DP> load;
  load.left = 0, load.page = -1;
  if (busy) load.start(p, walk.cur);
  const uint32_t ring = smem_u32(mine);
  auto refill = [&](int to) {
    if (walk.look_ahead(p, load.left)) load.start(p, walk.nxt);
    load.issue(p, ring + to * Tile::kStageBytes);
  };
#pragma unroll 1
  for (int i = 0; i < Cfg::kStages - 1; ++i) refill(i);

  AttnCursor at = walk.cur.at;
  bool begun = at.tile == at.r.t0, fresh = true;
  float m[H], l[H];
  float2 o[H][E / 2];
  int stage = 0;
  for (int i = 0; busy;) {
    const int kv = at.kv, h0 = at.blk * p.block_heads, nh = min(p.block_heads, p.group - h0);
    if (fresh) {
#pragma unroll
      for (int h = 0; h < H; ++h) {
        m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
        for (int e = 0; e < E / 2; ++e) o[h][e] = make_float2(0.f, 0.f);
      }
    }
    // an item's queries are a group of copies of their own; its first tile waits for all
    if (fresh)
      cp_async_wait<0>();
    else
      cp_async_wait<Cfg::kStages - 2>();
    fresh = false;
    __syncwarp();
    // the stage read in the last round is free again
    refill(stage == 0 ? Cfg::kStages - 1 : stage - 1);

    const unsigned char* ks = mine + stage * Tile::kStageBytes;
    const int tok = lane & 15, half = lane >> 4;
    float2 acc[H];
#pragma unroll
    for (int h = 0; h < H; ++h) acc[h] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int c = half * (p.c.dim / 8); c < (half + 1) * (p.c.dim / 8); ++c) {
      const float4 kf = *reinterpret_cast<const float4*>(ks + Tile::offset(tok, c));
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const float4 qv = *reinterpret_cast<const float4*>(sq + h * DP + c * N);
        acc[h] = fma2(make_float2(qv.x, qv.y), make_float2(kf.x, kf.y), acc[h]);
        acc[h] = fma2(make_float2(qv.z, qv.w), make_float2(kf.z, kf.w), acc[h]);
      }
    }
    const int at_pos = at.tile * kAttnTile + tok;
    const bool live = at_pos >= at.r.lo && at_pos < at.r.n;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const float half_sum = acc[h].x + acc[h].y;
      float x = half_sum + __shfl_xor_sync(0xffffffffu, half_sum, 16);
      x = live ? x * p.scale_log2 : -INFINITY;
      float mx = x;
#pragma unroll
      for (int d = 8; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float m2 = fmaxf(m[h], mx), base = m2 == -INFINITY ? 0.f : m2;
      const float keep = exp2_fast(m[h] - base), pr = exp2_fast(x - base);
      m[h] = m2;
      l[h] = l[h] * keep + (half ? 0.f : pr);  // per lane; added over the lanes at the item's end
      if (half == 0) sp[tok * H + h] = make_float2(pr, pr);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) o[h][e].x *= keep, o[h][e].y *= keep;
    }
    __syncwarp();
    const unsigned char* vs = ks + Tile::kTileBytes;
#pragma unroll 4
    for (int t = 0; t < kAttnTile; ++t) {
      float2 vf[E / 2];
#pragma unroll
      for (int e = 0; e < E; e += W) {  // elements W lane .. of every 32 W
        const unsigned char* from = vs + Tile::offset(t, (e * 32 + W * lane) / N) + (W * lane) % N * 4;
        if constexpr (W == 4) {
          const float4 v = *reinterpret_cast<const float4*>(from);
          vf[e / 2] = make_float2(v.x, v.y), vf[e / 2 + 1] = make_float2(v.z, v.w);
        } else {
          vf[e / 2] = *reinterpret_cast<const float2*>(from);
        }
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const float2 pr = sp[t * H + h];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) o[h][e] = fma2(pr, vf[e], o[h][e]);
      }
    }
    stage = stage + 1 == Cfg::kStages ? 0 : stage + 1;

    const bool done = at.tile + 1 == at.r.t1, end = i + 1 == walk.cur.count;
    if (done || end) {
      const AttnPlace to = attn_place<DP>(p, walk.list, walk.cur, at, i, begun, done, reinterpret_cast<float*>(mine), s_ml[warp]);
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int d = 16; d; d >>= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
        if (h >= nh) continue;
        const float f = to.whole ? (l[h] > 0.f ? 1.f / l[h] : (l[h] == 0.f ? 0.f : l[h])) : 1.f;  // NaN stays
        if (!to.whole && lane == 0) to.ml[h] = make_float2(m[h], l[h]);
        float* out = to.whole ? (float*)p.out + (((int64_t)at.row * p.c.kv_heads + kv) * p.group + h0 + h) * p.c.dim
                              : to.sums + h * to.pitch;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const int d = e / W * (32 * W) + W * lane + e % W;
          if (d < p.c.dim) *reinterpret_cast<float2*>(out + d) = make_float2(o[h][e / 2].x * f, o[h][e / 2].y * f);
        }
      }
      begun = true, fresh = true;
    }
    __syncwarp();
    if (end) {
      if (!walk.step()) break;
      at = walk.cur.at, i = 0;
      begun = at.tile == at.r.t0;
      load_q(at);
    } else {
      at.next(p), ++i;
      if (done) load_q(at);
    }
  }
  if (p.direct) attn_gather<float, Cfg::kWarps, H, DP>(p, attn_smem, Cfg::kWarpBytes, s_ml);
}

template <int DP, int NT>
struct AttnMmaCfg {
  using Tile = AttnTileCfg<2, DP>;
  static constexpr int kHeads = 8 * NT;            // query heads of a block
  static constexpr bool kQShared = NT * DP > 256;  // query fragments in shared memory, not registers
  static constexpr int kQBytes = kQShared ? kHeads * DP * 2 : 0;
  // heads of 64: tiles of half the bytes and nearly the instructions, so twice the warps
  static constexpr bool kMany = DP == 64 && NT == 1;
  static constexpr int kStages = DP == 256 ? 2 : (DP == 128 || kMany ? 3 : 6);
  static constexpr int kWarpBytes = kStages * Tile::kStageBytes + kQBytes;
  static constexpr int kFit = 220 * 1024 / kWarpBytes, kMost = kMany ? 16 : 8;
  static constexpr int kWarps = kFit < kMost ? kFit : kMost;
  static constexpr int kSmemBytes = 1024 + kWarps * kWarpBytes;  // aligned to 1024 bytes
};

// Tensor-core attention for 16-bit types, 8 * NT query heads at a time.  A tile's
// keys are the rows of S^T = K Q^T (m16n8k16: 16 tokens by 8 heads, so a group
// of up to eight heads fills the instruction), its values those of
// O^T += V^T P^T; both come from shared memory by ldmatrix, and P^T is S^T's own
// fragment, transposed in registers by movmatrix.
//
// Probabilities enter the second product as a 16-bit number and a 16-bit
// remainder: with the first alone the sums would be off by as much as the
// rounding of the result (1.7e-3 becomes 2.3e-3 of a bf16 output); the second
// costs one more instruction where memory is the bound.  In fp16 the largest
// probability stands as 2^15, here and in the sum that divides: next to 1 what lies
// below 2^-25 would be lost, and from the values alone (131071 tokens of 2^-26 are 0.2 %
// of the sum); so it is what lies below 2^-40.  An infinite value of a token that is attended to
// gives infinity or NaN.
//
// 256 rows of up to 4096 tokens, 32/8 heads of 128, bf16, 2.03 GB: 310 us with plan
// and join (6.5 TB/s), where the same kernel with a copy instruction a lane took 419;
// one row of 131072 tokens 100 us (5.4 TB/s).  Groups of 32 heads are bound by issue
// slots (2.1 TB/s).
template <bool BF16, int DP, int NT, bool TMA>
__global__ void __launch_bounds__(AttnMmaCfg<DP, NT>::kWarps * 32, 1)
    attn_mma_kernel(const AttnParams p, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
  using Cfg = AttnMmaCfg<DP, NT>;
  using Tile = AttnTileCfg<2, DP>;
  using T = typename Elem<BF16>::T;
  constexpr int KS = DP / 16, STAGES = Cfg::kStages;
  constexpr float kUnit = BF16 ? 1.f : 0x1p15f;  // what a probability of 1 stands as
  extern __shared__ __align__(128) unsigned char attn_smem[];
  __shared__ uint64_t bars[TMA ? Cfg::kWarps * STAGES : 1];
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float2 s_ml[Cfg::kWarps][Cfg::kHeads];
  unsigned char* rings = attn_smem + ((1024 - (smem_u32(attn_smem) & 1023)) & 1023);
  unsigned char* mine = rings + warp * Cfg::kWarpBytes;
  const uint32_t ring = smem_u32(mine), sq = ring + STAGES * Tile::kStageBytes;
  uint64_t* bar = bars + (TMA ? warp * STAGES : 0);
  if constexpr (TMA) {
    if (threadIdx.x == 0) abort_flag = 0;
    if (lane == 0) {
      for (int i = 0; i < STAGES; ++i) mbar_init(bar + i, 1);
      fence_barrier_init();
      prefetch_tmap(&mk);
      prefetch_tmap(&mv);
    }
  } else if (p.c.dim < DP) {  // columns that no copy fills
    for (int i = lane; i < STAGES * Tile::kStageBytes / 16; i += 32) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
  }
  if (lane < Cfg::kHeads) s_ml[warp][lane] = make_float2(-INFINITY, 0.f);
  if constexpr (TMA) __syncthreads();  // abort_flag
  __syncwarp();
  griddep_wait();
  griddep_launch();
  AttnWalk walk;
  const bool busy = walk.start(p);
  if (!busy && !p.direct) return;

  // the item's queries: B fragments in registers, or rows in shared memory (cp.async)
  uint32_t qf[Cfg::kQShared ? 1 : NT][Cfg::kQShared ? 1 : KS][2];
  auto load_q = [&](const AttnCursor& c) {
    const int h0 = c.blk * p.block_heads, nh = min(p.block_heads, p.group - h0);
    const T* q = (const T*)p.q + c.row * p.q_row + (c.kv * p.group + h0) * p.q_head;
    if constexpr (Cfg::kQShared) {
      for (int j = lane; j < Cfg::kHeads * Tile::kChunks; j += 32) {
        const int h = j / Tile::kChunks, c = j % Tile::kChunks;
        const bool ok = h < nh && c * 8 < p.c.dim;
        cp_async16_or_zero(sq + h * (DP * 2) + ((c ^ (h & 7)) << 4), ok ? q + h * p.q_head + c * 8 : q, ok);
      }
      cp_async_commit();
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + (lane >> 2);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int d = ks * 16 + j * 8 + (lane & 3) * 2;
            qf[nt][ks][j] = h < nh && d < p.c.dim ? *reinterpret_cast<const uint32_t*>(q + h * p.q_head + d) : 0u;
          }
      }
    }
  };
  if (busy) load_q(walk.cur.at);  // on their way while the first pages are looked up

  std::conditional_t<TMA, AttnTmaLoader<DP>, AttnCopyLoader<2, DP>> load;
  load.left = 0, load.page = -1;
  if (busy) load.start(p, walk.cur);
  int flying = 0;  // TMA: tiles whose copies have not been waited for
  auto refill = [&](int to) {
    if (walk.look_ahead(p, load.left)) load.start(p, walk.nxt);
    if constexpr (TMA) {
      flying += load.left > 0;
      load.issue(p, &mk, &mv, ring + to * Tile::kStageBytes, bar + to);
    } else {
      load.issue(p, ring + to * Tile::kStageBytes);
    }
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; ++i) refill(i);

  // ldmatrix rows of this lane: keys (token l & 15, chunk 2 ks + l / 16), values
  // transposed (token (l & 7) + 8 (l / 16), chunk 2 mt + (l / 8) % 2); four chunk
  // pairs make a block, so step j adds a block and one of four offsets
  const int krow = lane & 15, vrow = (lane & 7) + ((lane >> 4) << 3);
  uint32_t koff[4], voff[4], qoff[4];  // qoff: shared queries, head (l & 7) + 8 (l / 16), chunk 2 ks + (l / 8) % 2
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    qoff[j] = vrow * DP * 2 + (((2 * j + ((lane >> 3) & 1)) ^ (lane & 7)) << 4);
    koff[j] = Tile::offset(krow, 2 * j + (lane >> 4));
    voff[j] = Tile::kTileBytes + Tile::offset(vrow, 2 * j + ((lane >> 3) & 1));
  }
  AttnCursor at = walk.cur.at;
  bool begun = at.tile == at.r.t0, fresh = true;
  float m[NT][2], l[NT][2], o[NT][KS][4];
  int stage = 0;
  uint32_t parity = 0;
  for (int i = 0; busy;) {
    if (fresh) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < 2; ++j) m[nt][j] = -INFINITY, l[nt][j] = 0.f;
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[nt][mt][j] = 0.f;
      }
    }
    if constexpr (TMA) {
      refill(stage == 0 ? STAGES - 1 : stage - 1);  // read in the last round: free again
      if (!mbar_wait_warp(bar + stage, parity, &abort_flag)) {
        // the status is raised; let this warp's copies land before the CTA's memory goes
        for (; flying > 0; --flying) {
          mbar_drain(bar + stage, parity);
          if (++stage == STAGES) stage = 0, parity ^= 1;
        }
        break;
      }
      --flying;
      if (Cfg::kQShared && fresh) {
        cp_async_wait<0>();
        __syncwarp();
      }
    } else {
      // an item's queries are a group of their own among the tiles'; the first of its tiles waits for all
      if (Cfg::kQShared && fresh)
        cp_async_wait<0>();
      else
        cp_async_wait<STAGES - 2>();
      __syncwarp();
      refill(stage == 0 ? STAGES - 1 : stage - 1);
    }
    fresh = false;
    const uint32_t base = ring + stage * Tile::kStageBytes;
    const bool inner = at.tile * kAttnTile >= at.r.lo && (at.tile + 1) * kAttnTile <= at.r.n;
    if (TMA && !inner) {
      // the copy brought whole pages: values outside the row's tokens must not
      // meet a zero probability as NaN or infinity
      for (int j = lane; j < kAttnTile * Tile::kChunks; j += 32) {
        const int row = j / Tile::kChunks, ps = at.tile * kAttnTile + row;
        if (ps < at.r.lo || ps >= at.r.n)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + Tile::kTileBytes +
                                                                       Tile::offset(row, j % Tile::kChunks)),
                       "r"(0)
                       : "memory");
      }
      fence_proxy_async_smem();  // before a later copy lands here
      __syncwarp();
    }

    float sc[NT][2][4];  // two chains of sums, even and odd steps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[nt][0][j] = sc[nt][1][j] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (!TMA && ks * 16 >= p.c.dim) break;
      uint32_t a[4];
      ldsm_x4(base + koff[ks & 3] + (ks >> 2) * (kAttnTile * 128), a);
      if constexpr (Cfg::kQShared) {
        static_assert(!Cfg::kQShared || NT % 2 == 0, "two groups of eight heads at a time");
#pragma unroll
        for (int nt = 0; nt < NT; nt += 2) {
          uint32_t b[4];
          ldsm_x4(sq + qoff[ks & 3] + nt * 8 * DP * 2 + (ks >> 2) * 128, b);
          mma_16816<BF16>(sc[nt][ks & 1], a, b[0], b[1]);
          mma_16816<BF16>(sc[nt + 1][ks & 1], a, b[2], b[3]);
        }
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816<BF16>(sc[nt][ks & 1], a, qf[nt][ks][0], qf[nt][ks][1]);
      }
    }
    const int p0 = at.tile * kAttnTile + (lane >> 2);  // this lane's tokens: p0, p0 + 8
    const bool live0 = inner || (p0 >= at.r.lo && p0 < at.r.n), live1 = inner || (p0 + 8 >= at.r.lo && p0 + 8 < at.r.n);
    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[4], keep[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = (sc[nt][0][j] + sc[nt][1][j]) * p.scale_log2;
        if (!(j < 2 ? live0 : live1)) x[j] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // the lane's two heads
        float mx = fmaxf(x[j], x[j + 2]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float m2 = fmaxf(m[nt][j], mx), top = m2 == -INFINITY ? 0.f : m2;
        keep[j] = exp2_fast(m[nt][j] - top);
        m[nt][j] = m2;
        x[j] = exp2_fast(x[j] - top) * kUnit;
        x[j + 2] = exp2_fast(x[j + 2] - top) * kUnit;
        l[nt][j] = l[nt][j] * keep[j] + x[j] + x[j + 2];  // of this lane's tokens; added over lanes at the end
      }
      if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[nt][mt][j] *= keep[j & 1];
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t w = pack2<BF16>(x[2 * j], x[2 * j + 1]);
        const float r0 = x[2 * j] - Elem<BF16>::to_f((uint16_t)w), r1 = x[2 * j + 1] - Elem<BF16>::to_f((uint16_t)(w >> 16));
        hi[nt][j] = movmatrix_t(w);
        lo[nt][j] = movmatrix_t(pack2<BF16>(r0, r1));
      }
    }
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) {
      if (!TMA && mt * 16 >= p.c.dim) break;
      uint32_t a[4];
      ldsm_x4_trans(base + voff[mt & 3] + (mt >> 2) * (kAttnTile * 128), a);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_16816<BF16>(o[nt][mt], a, hi[nt][0], hi[nt][1]);
        mma_16816<BF16>(o[nt][mt], a, lo[nt][0], lo[nt][1]);
      }
    }
    if (++stage == STAGES) stage = 0, parity ^= 1;

    const bool done = at.tile + 1 == at.r.t1, end = i + 1 == walk.cur.count;
    const AttnCursor was = at;
    if (!end) {
      at.next(p);
      if (done) {  // the next item's queries, on their way while this one's sums are written
        __syncwarp();
        load_q(at);
      }
    }
    if (done || end) {
      const AttnPlace to = attn_place<DP>(p, walk.list, walk.cur, was, i, begun, done, reinterpret_cast<float*>(mine),
                                          s_ml[warp]);
      const int h0 = was.blk * p.block_heads, nh = min(p.block_heads, p.group - h0);
      const int64_t head0 = ((int64_t)was.row * p.c.kv_heads + was.kv) * p.group + h0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float sum = l[nt][j];
          sum += __shfl_xor_sync(0xffffffffu, sum, 4);
          sum += __shfl_xor_sync(0xffffffffu, sum, 8);
          sum += __shfl_xor_sync(0xffffffffu, sum, 16);
          const int h = nt * 8 + (lane & 3) * 2 + j;
          if (h >= nh) continue;
          const float f = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // NaN stays
          if (!to.whole && lane < 4) to.ml[h] = make_float2(m[nt][j], sum);
          T* out = (T*)p.out + (head0 + h) * p.c.dim;
          float* part = to.sums + h * to.pitch;
#pragma unroll
          for (int mt = 0; mt < KS; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = mt * 16 + e * 8 + (lane >> 2);
              if (d >= p.c.dim) continue;
              if (to.whole)
                out[d] = Chunk<T>::put(o[nt][mt][2 * e + j] * f);
              else
                part[d] = o[nt][mt][2 * e + j];
            }
        }
      }
      begun = true, fresh = true;
    }
    __syncwarp();
    ++i;
    if (end) {
      if (!walk.step()) break;
      at = walk.cur.at, i = 0;
      begun = at.tile == at.r.t0;
      load_q(at);
    }
  }
  if (p.direct) attn_gather<T, Cfg::kWarps, Cfg::kHeads, DP>(p, rings, Cfg::kWarpBytes, s_ml);
}

// Joins the parts of the items that segments cut.  Of an item of up to 32 parts a
// warp takes a head, one part after the other; of more parts, a CTA takes 32
// elements of a head, each warp a run of parts, four of them at a time.  Bound by
// the latency of the L2: 9 us for 8 items of 370 parts, 13 us for 1700 of 2 to 18,
// against 35 us with a load behind each branch.
constexpr int kJoinWarps = 8, kJoinGrid = 3 * 148, kJoinSlice = 32;

// Sums of one head of an item from its parts; a lane holds four elements.
struct AttnSum {
  float m, l, o[4];
  __device__ __forceinline__ void clear() { m = -INFINITY, l = o[0] = o[1] = o[2] = o[3] = 0.f; }
  // Parts [i0, i1) of item `c`, head h, elements e0 + 4 (lane % LANES): 32 / LANES
  // parts at a time, whose sums the lanes of one element keep apart.  Warp-collective.
  template <int LANES>
  __device__ __forceinline__ void add(const AttnParams& p, const int4& c, int h, int i0, int i1, int e0) {
    constexpr int PER = 32 / LANES;
    const int lane = threadIdx.x & 31, dim = p.c.dim;
    const int e = min(e0 + lane % LANES * 4, dim - 4);  // lanes past dim repeat its last four
    for (int first = i0; first < i1; first += 32) {
      const int n = min(32, i1 - first), i = first + lane;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (lane < n) ml = p.part_ml[((c.z + i) * 2ll + (i == 0 ? 1 : 0)) * p.block_heads + h];
      // eight loads at a time, none behind a branch: one from the L2 takes longer
      // than all the arithmetic
      float4 v[8];
      auto load = [&](int j0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at = first + min(j0 + j * PER + lane / LANES, n - 1);
          v[j] = *reinterpret_cast<const float4*>(
              p.part_o + (((c.z + at) * 2ll + (at == 0 ? 1 : 0)) * p.block_heads + h) * dim + e);
        }
      };
      load(0);
      float top = ml.x;
#pragma unroll
      for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      top = fmaxf(top, m);
      const float base = top == -INFINITY ? 0.f : top;
      const float keep = exp2_fast(m - base), f = exp2_fast(ml.x - base);
      float sum = ml.y * f;
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      m = top, l = l * keep + sum;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] *= keep;
      for (int j0 = 0;;) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int at = j0 + j * PER + lane / LANES;
          const float g = __shfl_sync(0xffffffffu, f, at & 31);
          if (at < n) o[0] += v[j].x * g, o[1] += v[j].y * g, o[2] += v[j].z * g, o[3] += v[j].w * g;
        }
        j0 += 8 * PER;
        if (j0 >= n) break;
        load(j0);
      }
    }
#pragma unroll
    for (int d = LANES; d < 32; d <<= 1)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] += __shfl_xor_sync(0xffffffffu, o[k], d);
  }
};

template <typename T>
__device__ __forceinline__ void join_put(const AttnParams& p, const int4& c, int h, int e, float l, const float* o) {
  const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays
  const int kv = c.y / p.blocks, h0 = (c.y - kv * p.blocks) * p.block_heads;
  T* out = (T*)p.out + (((int64_t)c.x * p.c.kv_heads + kv) * p.group + h0 + h) * p.c.dim + e;
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = Chunk<T>::put(o[j] * f);
}

template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const AttnParams p) {
  __shared__ float s_o[kJoinWarps][kJoinSlice];
  __shared__ float2 s_ml[kJoinWarps];
  griddep_wait();
  griddep_launch();
  const int near = p.work->cuts[0], far = p.work->cuts[1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = p.c.dim, bh = p.block_heads;
  auto heads_of = [&](const int4& c) { return min(bh, p.group - c.y % p.blocks * bh); };
  AttnSum a;
  const int slices = (dim + kJoinSlice - 1) / kJoinSlice;
  for (int t = blockIdx.x; t < far * bh * slices; t += gridDim.x) {
    const int4 c = p.cut[p.cut_room - 1 - t / (bh * slices)];
    const int h = t / slices % bh, e0 = t % slices * kJoinSlice;
    if (h >= heads_of(c)) continue;
    a.clear();
    a.add<kJoinSlice / 4>(p, c, h, c.w * warp / kJoinWarps, c.w * (warp + 1) / kJoinWarps, e0);
    __syncthreads();  // the slice before has been read
    if (lane < kJoinSlice / 4) *reinterpret_cast<float4*>(&s_o[warp][lane * 4]) = make_float4(a.o[0], a.o[1], a.o[2], a.o[3]);
    if (lane == 0) s_ml[warp] = make_float2(a.m, a.l);
    __syncthreads();
    const int e = threadIdx.x * 4;
    if (e < kJoinSlice && e0 + e < dim) {
      float top = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, s_ml[w].x);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        const float f = exp2_fast(s_ml[w].x - base);
        l += s_ml[w].y * f;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += s_o[w][e + j] * f;
      }
      join_put<T>(p, c, h, e0 + e, l, o);
    }
  }
  const int halves = (dim + 127) / 128;
  for (int t = warp * gridDim.x + blockIdx.x; t < near * bh * halves; t += gridDim.x * kJoinWarps) {
    const int4 c = p.cut[t / (bh * halves)];
    const int h = t / halves % bh, e0 = t % halves * 128;
    if (h >= heads_of(c)) continue;
    a.clear();
    a.add<32>(p, c, h, 0, c.w, e0);
    if (e0 + lane * 4 < dim) join_put<T>(p, c, h, e0 + lane * 4, a.l, a.o);
  }
}

}  // namespace plora
