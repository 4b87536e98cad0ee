// Paged key-value cache: appending new tokens with their position rotation,
// and attention of one new token per row over the cache.
//
// Cache layout: k and v are (num_pages, kv_heads, page_size, head_dim), so the
// tokens of one head in one page are one contiguous run; a row's tokens are
// found through its page table, position p at slot p % page_size of page
// table[p / page_size].
#pragma once

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
// cosines of a token are computed once and shared by all of its heads.
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
// there: an item is a row and a key-value head (or a block of its query
// heads), a tile 16 of its tokens, and the tiles of all items in order are
// dealt in equal contiguous shares to the grid's warps, each of which streams
// its share through a ring of shared-memory stages of its own (no barrier
// between warps).  An item cut by the ends of shares is put together in two
// steps: first the parts of a CTA's warps, then, by attn_join_kernel, what the
// CTAs left in the workspace, always in the order of the shares.  Every item has
// at least one (empty) tile, so rows without tokens are written too.
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
  // workspace.  A part of an item: its sums of block_heads heads, and for each
  // head its maximum (in units of scale_log2) and sum of probabilities
  float* warp_o;   // (warps, block_heads, dim): a warp's part of the item that another began
  float* cta_o;    // (CTAs, 2, block_heads, dim): a CTA's parts of the items that it shares (0: begun by
  float2* cta_ml;  // (CTAs, 2, block_heads)       another, 1: begun here)
  int4* desc;      // (CTAs): row, kv head, head block, CTAs of the item begun here and shared (0: none)
};

struct AttnRow {
  int lo, n;   // tokens [lo, n)
  int t0, t1;  // tiles [t0, t1), at least one
};
__device__ __forceinline__ AttnRow attn_row(const AttnParams& p, int row) {
  AttnRow r;
  int64_t n = p.seq_lens[row];
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
  AttnRow r;
  __device__ __forceinline__ void next(const AttnParams& p) {
    if (++tile < r.t1) return;
    if (++blk == p.blocks) {
      blk = 0;
      if (++kv == p.c.kv_heads) {
        kv = 0;
        if (++row < p.rows) r = attn_row(p, row);
      }
    }
    tile = r.t0;
  }
};

struct AttnShare {
  int64_t begin;  // first tile of this warp in the list
  int count;      // its tiles
  int warps;      // warps with a share, of all CTAs; warp w of CTA c is number c * WARPS + w
  int base, rem;  // the first rem of them have base + 1 tiles, the others base
  AttnCursor at;  // at `begin`
  // The warp whose share holds tile x of the list.
  __device__ __forceinline__ int holder(int64_t x) const {
    const int64_t split = (int64_t)rem * (base + 1);
    return x < split ? (int)(x / (base + 1)) : rem + (int)((x - split) / base);
  }
};

// Sum over the CTA's threads before this one (exclusive) and over all of them.
template <int WARPS>
__device__ __forceinline__ int block_scan(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += u;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += s_warp[w];
    sum += s_warp[w];
  }
  *total = sum;
  return before + incl - v;
}

// The calling warp's share.  Block-collective; warps without one get count 0.
template <int WARPS>
__device__ __forceinline__ AttnShare attn_share(const AttnParams& p) {
  constexpr int THREADS = WARPS * 32;
  __shared__ int s_warp[WARPS];
  __shared__ int s_row[WARPS];
  __shared__ int64_t s_before[WARPS], s_begin[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5;
  const int per_row = p.c.kv_heads * p.blocks;
  auto tiles_of = [&](int row) {
    if (row >= p.rows) return 0;
    const AttnRow r = attn_row(p, row);
    return r.t1 - r.t0;
  };
  // tiles of the rows before this thread's (of the last round), and of all
  int n = tiles_of(tid), sum;
  int64_t mine = block_scan<WARPS>(n, s_warp, &sum), tiles = sum;
  for (int first = THREADS; first < p.rows; first += THREADS) {
    block_scan<WARPS>(tiles_of(first + tid), s_warp, &sum);
    tiles += sum;
  }
  const int64_t total = tiles * per_row;
  AttnShare s;
  const int all = gridDim.x * WARPS, id = blockIdx.x * WARPS + warp;
  s.warps = total < all ? (int)total : all;
  if (total <= INT32_MAX) {  // a 64-bit division takes a microsecond's tenth
    s.base = (int)((uint32_t)total / (uint32_t)s.warps);
    s.rem = (int)((uint32_t)total - (uint32_t)s.base * s.warps);
  } else {
    s.base = (int)(total / s.warps);
    s.rem = (int)(total - (int64_t)s.base * s.warps);
  }
  s.begin = (int64_t)id * s.base + min(id, s.rem);
  s.count = id < s.warps ? s.base + (id < s.rem ? 1 : 0) : 0;
  if ((tid & 31) == 0) s_begin[warp] = s.count ? s.begin : -1;
  __syncthreads();
  int64_t before = 0;  // tiles of the rounds before
  for (int first = 0;;) {
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const int64_t x = s_begin[w];
      if (x >= mine * per_row && x < (mine + n) * per_row) {
        s_row[w] = first + tid;
        s_before[w] = mine;
      }
    }
    if (p.rows <= THREADS) break;
    block_scan<WARPS>(n, s_warp, &sum);
    before += sum;
    first += THREADS;
    if (first >= p.rows) break;
    n = tiles_of(first + tid);
    mine = before + block_scan<WARPS>(n, s_warp, &sum);
  }
  __syncthreads();
  if (s.count) {
    s.at.row = s_row[warp];
    s.at.r = attn_row(p, s.at.row);
    const int nt = s.at.r.t1 - s.at.r.t0;
    const int rest = (int)(s.begin - s_before[warp] * per_row);
    const int item = rest / nt;
    s.at.kv = item / p.blocks;
    s.at.blk = item - s.at.kv * p.blocks;
    s.at.tile = s.at.r.t0 + rest - item * nt;
  }
  return s;
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
  int page, inner;  // of this lane's token of tile `at`; page -1: reads as zeros

  __device__ __forceinline__ void look_up(const AttnParams& p) {
    page = -1, inner = 0;
    if (left <= 0) return;
    const int pos = at.tile * kAttnTile + (threadIdx.x & 15);
    if (pos >= at.r.lo && pos < at.r.n) {
      const int e = p.c.page.div(pos);
      page = p.c.table[at.row * p.c.table_stride + e];
      if ((uint32_t)page >= (uint32_t)p.c.num_pages) {
        raise_status(PLORA_DEV_PAGE_RANGE);
        page = -1;
      }
      inner = (at.kv * p.c.page_size + pos - e * p.c.page_size) * p.c.dim;
    }
  }
  // Starts the copies of tile `at` (none past the share's end) and steps on.
  __device__ __forceinline__ void issue(const AttnParams& p, uint32_t stage) {
    if (left > 0) {
      constexpr int LANES = Tile::kChunks < 32 ? Tile::kChunks : 32;  // lanes of a row
      const int lane = threadIdx.x & 31, lc = lane % LANES;
#pragma unroll
      for (int r0 = 0; r0 < kAttnTile; r0 += 32 / LANES) {
        const int row = r0 + lane / LANES;
        const int pg = __shfl_sync(0xffffffffu, page, row), in = __shfl_sync(0xffffffffu, inner, row);
        const bool ok = pg >= 0;
        const char* k = (const char*)p.c.k + (ok ? (pg * p.c.k_page + in) * EB : 0);
        const char* v = (const char*)p.c.v + (ok ? (pg * p.c.v_page + in) * EB : 0);
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
  // One lane's: starts the copies of tile `at`, completing on `bar`, and steps on.
  __device__ __forceinline__ void issue(const AttnParams& p, const CUtensorMap* mk, const CUtensorMap* mv,
                                        uint32_t stage, uint64_t* bar) {
    if (left <= 0) return;
    mbar_arrive_expect_tx(bar, Tile::kStageBytes);
    tma_load_tile(stage, mk, bar, slot, at.kv, page);
    tma_load_tile(stage + Tile::kTileBytes, mv, bar, slot, at.kv, page);
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

// What the warps of a CTA leave to one another: parts of items cut by the ends
// of shares, slot 0 of the item that another warp began, slot 1 of the one that
// goes on in the next warp.  The sums of a warp's last part lie in its ring (rows of
// DP + 4 floats: fragment rows then fall into different banks), those of an
// earlier one, while the ring is still in use, in the workspace.
template <int WARPS, int HEADS>
struct AttnBoard {
  float2 ml[WARPS][2][HEADS];  // maximum, sum
  int4 item[WARPS][2];         // row, kv head, head block; w: 0 none, 1 in the workspace, 2 in the ring
  int done[WARPS];             // the item of slot 0 ends in this warp
  int ctas[WARPS];             // CTAs of the item of slot 1
};

// Where a warp puts the sums of an item that it has done its part of.
struct AttnPlace {
  bool whole;   // to the output
  int slot;
  float* sums;  // else here, rows of `pitch`
  int pitch;
};
template <int WARPS, int HEADS, int DP>
__device__ __forceinline__ AttnPlace attn_place(const AttnParams& p, const AttnShare& s, AttnBoard<WARPS, HEADS>& board,
                                                float* ring, const AttnCursor& at, int i, bool begun, bool done) {
  const int warp = threadIdx.x >> 5;
  AttnPlace o;
  o.whole = begun && done;
  o.slot = begun ? 1 : 0;
  const bool last = i + 1 == s.count;
  o.sums = last ? ring : p.warp_o + (int64_t)(blockIdx.x * WARPS + warp) * p.block_heads * p.c.dim;
  o.pitch = last ? DP + 4 : p.c.dim;
  if (!o.whole && (threadIdx.x & 31) == 0) {
    board.item[warp][o.slot] = make_int4(at.row, at.kv, at.blk, last ? 2 : 1);
    if (begun)  // its last tile is this many on
      board.ctas[warp] = s.holder(s.begin + i + (at.r.t1 - 1 - at.tile)) / WARPS - blockIdx.x + 1;
    else
      board.done[warp] = done;
  }
  return o;
}

// Four elements of a head from its parts' maxima, sums and elements.
struct AttnSum {
  float m, l, o[4];
  __device__ __forceinline__ void clear() { m = -INFINITY, l = o[0] = o[1] = o[2] = o[3] = 0.f; }
  __device__ __forceinline__ void add(float pm, float pl, const float4& v) {
    const float m2 = fmaxf(m, pm), top = m2 == -INFINITY ? 0.f : m2;
    const float keep = exp2_fast(m - top), f = exp2_fast(pm - top);
    m = m2;
    l = l * keep + pl * f;
    o[0] = o[0] * keep + v.x * f, o[1] = o[1] * keep + v.y * f, o[2] = o[2] * keep + v.z * f, o[3] = o[3] * keep + v.w * f;
  }
  template <typename T>
  __device__ __forceinline__ void put(T* out) const {
    const float f = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = Chunk<T>::put(o[e] * f);
  }
};

// Puts the warps' parts together: a chain is the parts of one item in
// neighbouring warps; a whole item goes to the output, else its sums go to the
// workspace for attn_join_kernel.  Block-collective; a warp takes a chain's head,
// a lane four (of 128) elements of it.
template <typename T, int WARPS, int HEADS, int DP>
__device__ __forceinline__ void attn_merge(const AttnParams& p, const AttnBoard<WARPS, HEADS>& board,
                                           const unsigned char* ring0, int ring_pitch) {
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = p.c.dim;
  int task = 0;
  bool shared = false;  // an item begun here goes on in the next CTA
  for (int w0 = -1; w0 < WARPS; ++w0) {  // chains: slot 0 of warp 0 (w0 = -1), slot 1 of warp w0
    const int w = max(w0, 0), slot = w0 < 0 ? 0 : 1;
    const int4 item = board.item[w][slot];
    if (item.w == 0) continue;
    int end = w + 1;  // past the chain's last warp
    bool closed = slot == 0 && board.done[0];
    while (!closed && end < WARPS && board.item[end][0].w) closed = board.done[end++];
    const bool whole = closed && slot == 1;
    const int h0 = item.z * p.block_heads, nh = min(p.block_heads, p.group - h0);
    if (slot == 1 && !closed) {
      shared = true;
      if (threadIdx.x == 0) p.desc[blockIdx.x] = make_int4(item.x, item.y, item.z, board.ctas[w]);
    }
    for (int h = 0; h < nh; ++h, ++task) {
      if (task % WARPS != warp) continue;
#pragma unroll
      for (int d0 = 0; d0 < DP; d0 += 128) {
        const int d = d0 + lane * 4;
        if (d >= dim) continue;
        AttnSum sum;
        sum.clear();
#pragma unroll 4
        for (int u = w; u < end; ++u) {
          const int sl = u == w ? slot : 0;
          const bool in_ring = board.item[u][sl].w == 2;
          const float* from = in_ring ? reinterpret_cast<const float*>(ring0 + u * ring_pitch) + h * (DP + 4)
                                      : p.warp_o + ((int64_t)(blockIdx.x * WARPS + u) * p.block_heads + h) * dim;
          const float2 ml = board.ml[u][sl][h];
          sum.add(ml.x, ml.y, *reinterpret_cast<const float4*>(from + d));
        }
        if (whole) {
          sum.put((T*)p.out + (((int64_t)item.x * p.c.kv_heads + item.y) * p.group + h0 + h) * dim + d);
        } else {
          const int64_t part = (blockIdx.x * 2ll + slot) * p.block_heads + h;
          *reinterpret_cast<float4*>(p.cta_o + part * dim + d) = make_float4(sum.o[0], sum.o[1], sum.o[2], sum.o[3]);
          if (d == 0) p.cta_ml[part] = make_float2(sum.m, sum.l);
        }
      }
    }
  }
  if (!shared && threadIdx.x == 0) p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
}

template <int DP>
struct AttnSimtCfg {
  using Tile = AttnTileCfg<4, DP>;
  static constexpr int kHeads = 8;  // query heads of a block
  static constexpr int kStages = DP == 256 ? 2 : 3;
  static constexpr int kWarps = DP == 256 ? 3 : (DP == 128 ? 4 : 8);
  static constexpr int kQBytes = kHeads * DP * 4, kPBytes = kAttnTile * kHeads * 4;
  static constexpr int kWarpBytes = kStages * Tile::kStageBytes + kQBytes + kPBytes;
  static constexpr int kSmemBytes = kWarps * kWarpBytes;
};

// CUDA-core attention for fp32 (TF32 products would lose 13 bits of it).
// Scores: lanes l and l + 16 take token l & 15, each half of the head's
// elements.  Sums: a lane owns DP / 32 elements of all heads.
template <int DP>
__global__ void __launch_bounds__(AttnSimtCfg<DP>::kWarps * 32, 1) attn_simt_kernel(const AttnParams p) {
  using T = float;
  using Cfg = AttnSimtCfg<DP>;
  using Tile = AttnTileCfg<4, DP>;
  constexpr int H = Cfg::kHeads, N = Chunk<T>::N, E = DP / 32;
  extern __shared__ __align__(128) unsigned char attn_smem[];
  __shared__ AttnBoard<Cfg::kWarps, H> board;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* mine = attn_smem + warp * Cfg::kWarpBytes;
  float* sq = reinterpret_cast<float*>(mine + Cfg::kStages * Tile::kStageBytes);  // [H][DP]
  float* sp = sq + H * DP;                                                        // [16][H]
  for (int i = lane; i < Cfg::kWarpBytes / 16; i += 32) reinterpret_cast<uint4*>(mine)[i] = make_uint4(0, 0, 0, 0);
  if (lane < 2) board.item[warp][lane].w = 0;
  griddep_wait();
  griddep_launch();
  const AttnShare s = attn_share<Cfg::kWarps>(p);
  __syncwarp();

  AttnCopyLoader<4, DP> load;
  load.at = s.at;
  load.left = s.count;
  if (s.count) load.look_up(p);
  const uint32_t ring = smem_u32(mine);
#pragma unroll
  for (int i = 0; i < Cfg::kStages - 1; ++i) load.issue(p, ring + i * Tile::kStageBytes);

  AttnCursor at = s.at;
  bool begun = at.tile == at.r.t0, fresh = true;
  float m[H], l[H], o[H][E];
  int stage = 0;
  for (int i = 0; i < s.count; ++i) {
    const int kv = at.kv, h0 = at.blk * p.block_heads, nh = min(p.block_heads, p.group - h0);
    if (fresh) {
      const T* q = (const T*)p.q + at.row * p.q_row + (kv * p.group + h0) * p.q_head;
      for (int h = 0; h < H; ++h)
        for (int d = lane; d < p.c.dim; d += 32) sq[h * DP + d] = h < nh ? Chunk<T>::get(q[h * p.q_head + d]) * p.scale_log2 : 0.f;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[h][e] = 0.f;
      }
      fresh = false;
    }
    cp_async_wait<Cfg::kStages - 2>();
    __syncwarp();
    // the stage read in the last round is free again
    const int ahead = stage == 0 ? Cfg::kStages - 1 : stage - 1;
    load.issue(p, ring + ahead * Tile::kStageBytes);

    const unsigned char* ks = mine + stage * Tile::kStageBytes;
    const int tok = lane & 15, half = lane >> 4;
    float acc[H];
#pragma unroll
    for (int h = 0; h < H; ++h) acc[h] = 0.f;
#pragma unroll 4
    for (int c = half * (Tile::kChunks / 2); c < (half + 1) * (Tile::kChunks / 2); ++c) {
      float kf[N];
      Chunk<T>::load(*reinterpret_cast<const uint4*>(ks + Tile::offset(tok, c)), kf);
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
          const float4 qv = *reinterpret_cast<const float4*>(sq + h * DP + c * N + j);
          acc[h] = fmaf(qv.x, kf[j], fmaf(qv.y, kf[j + 1], fmaf(qv.z, kf[j + 2], fmaf(qv.w, kf[j + 3], acc[h]))));
        }
      }
    }
    const int at_pos = at.tile * kAttnTile + tok;
    const bool live = at_pos >= at.r.lo && at_pos < at.r.n;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      float x = acc[h] + __shfl_xor_sync(0xffffffffu, acc[h], 16);
      x = live ? x : -INFINITY;
      float mx = x;
#pragma unroll
      for (int d = 8; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float m2 = fmaxf(m[h], mx), base = m2 == -INFINITY ? 0.f : m2;
      const float keep = exp2_fast(m[h] - base), pr = exp2_fast(x - base);
      m[h] = m2;
      l[h] = l[h] * keep + (half ? 0.f : pr);  // per lane; added over the lanes at the item's end
      if (half == 0) sp[tok * H + h] = pr;
#pragma unroll
      for (int e = 0; e < E; ++e) o[h][e] *= keep;
    }
    __syncwarp();
    const unsigned char* vs = ks + Tile::kTileBytes;
#pragma unroll 2
    for (int t = 0; t < kAttnTile; ++t) {
      float vf[E];
#pragma unroll
      for (int e = 0; e < E; e += 2) {  // elements 2 lane, 2 lane + 1 of every 64
        const int d = e * 32 + 2 * lane;
        const T* src = reinterpret_cast<const T*>(vs + Tile::offset(t, d / N)) + d % N;
        vf[e] = Chunk<T>::get(src[0]), vf[e + 1] = Chunk<T>::get(src[1]);
      }
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const float pr = sp[t * H + h];
#pragma unroll
        for (int e = 0; e < E; ++e) o[h][e] = fmaf(pr, vf[e], o[h][e]);
      }
    }
    stage = stage + 1 == Cfg::kStages ? 0 : stage + 1;

    const bool done = at.tile + 1 == at.r.t1;
    if (done || i + 1 == s.count) {
      __syncwarp();  // the ring may take the sums
      const AttnPlace to = attn_place<Cfg::kWarps, H, DP>(p, s, board, reinterpret_cast<float*>(mine), at, i, begun, done);
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int d = 16; d; d >>= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
        if (h >= nh) continue;
        const float f = l[h] > 0.f ? 1.f / l[h] : (l[h] == 0.f ? 0.f : l[h]);  // NaN stays
        if (!to.whole && lane == 0) board.ml[warp][to.slot][h] = make_float2(m[h], l[h]);
        float* out = to.whole ? (float*)p.out + (((int64_t)at.row * p.c.kv_heads + kv) * p.group + h0 + h) * p.c.dim
                              : to.sums + h * to.pitch;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const int d = e * 32 + 2 * lane;
          if (d < p.c.dim) *reinterpret_cast<float2*>(out + d) = to.whole ? make_float2(o[h][e] * f, o[h][e + 1] * f)
                                                                          : make_float2(o[h][e], o[h][e + 1]);
        }
      }
      begun = true, fresh = true;
    }
    at.next(p);
    __syncwarp();
  }
  attn_merge<float, Cfg::kWarps, H, DP>(p, board, attn_smem, Cfg::kWarpBytes);
}

template <int DP, int NT>
struct AttnMmaCfg {
  using Tile = AttnTileCfg<2, DP>;
  static constexpr int kHeads = 8 * NT;            // query heads of a block
  static constexpr bool kQShared = NT * DP > 256;  // query fragments in shared memory, not registers
  static constexpr int kQBytes = kQShared ? kHeads * DP * 2 : 0;
  static constexpr int kStages = DP == 256 ? 2 : (DP == 128 ? 3 : 6);
  static constexpr int kWarpBytes = kStages * Tile::kStageBytes + kQBytes;
  static constexpr int kFit = 220 * 1024 / kWarpBytes;
  static constexpr int kWarps = kFit < 8 ? kFit : 8;
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
// costs one more instruction where memory is the bound.
template <bool BF16, int DP, int NT, bool TMA>
__global__ void __launch_bounds__(AttnMmaCfg<DP, NT>::kWarps * 32, 1)
    attn_mma_kernel(const AttnParams p, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
  using Cfg = AttnMmaCfg<DP, NT>;
  using Tile = AttnTileCfg<2, DP>;
  using T = typename Elem<BF16>::T;
  constexpr int KS = DP / 16, STAGES = Cfg::kStages;
  extern __shared__ __align__(128) unsigned char attn_smem[];
  __shared__ uint64_t bars[TMA ? Cfg::kWarps * STAGES : 1];
  __shared__ int abort_flag;
  __shared__ AttnBoard<Cfg::kWarps, Cfg::kHeads> board;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  if (lane < 2) board.item[warp][lane].w = 0;
  griddep_wait();
  griddep_launch();
  const AttnShare s = attn_share<Cfg::kWarps>(p);
  __syncwarp();

  AttnCopyLoader<2, DP> copy;
  AttnTmaLoader<DP> tma;
  if constexpr (TMA) {
    tma.at = s.at, tma.left = s.count;
    if (lane == 0 && s.count) {
      tma.look_up(p);
#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) tma.issue(p, &mk, &mv, ring + i * Tile::kStageBytes, bar + i);
    }
  } else {
    copy.at = s.at, copy.left = s.count;
    if (s.count) copy.look_up(p);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) copy.issue(p, ring + i * Tile::kStageBytes);
  }

  // ldmatrix rows of this lane: keys (token l & 15, chunk 2 ks + l / 16), values
  // transposed (token (l & 7) + 8 (l / 16), chunk 2 mt + (l / 8) % 2); four chunk
  // pairs make a block, so step j adds a block and one of four offsets
  const int krow = lane & 15, vrow = (lane & 7) + ((lane >> 4) << 3);
  uint32_t koff[4], voff[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    koff[j] = Tile::offset(krow, 2 * j + (lane >> 4));
    voff[j] = Tile::kTileBytes + Tile::offset(vrow, 2 * j + ((lane >> 3) & 1));
  }
  AttnCursor at = s.at;
  bool begun = at.tile == at.r.t0, fresh = true;
  uint32_t qf[Cfg::kQShared ? 1 : NT][Cfg::kQShared ? 1 : KS][2];
  float m[NT][2], l[NT][2], o[NT][KS][4];
  int stage = 0;
  uint32_t parity = 0;
  for (int i = 0; i < s.count; ++i) {
    if (fresh) {
      const int h0 = at.blk * p.block_heads, nh = min(p.block_heads, p.group - h0);
      const T* q = (const T*)p.q + at.row * p.q_row + (at.kv * p.group + h0) * p.q_head;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (Cfg::kQShared) {
          for (int j = lane; j < 8 * Tile::kChunks; j += 32) {
            const int h = nt * 8 + j / Tile::kChunks, c = j % Tile::kChunks;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (h < nh && c * 8 < p.c.dim) u = *reinterpret_cast<const uint4*>(q + h * p.q_head + c * 8);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sq + h * (DP * 2) + ((c ^ (h & 7)) << 4)),
                         "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w)
                         : "memory");
          }
        } else {
          const int h = nt * 8 + (lane >> 2);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int d = ks * 16 + j * 8 + (lane & 3) * 2;
              qf[nt][ks][j] = h < nh && d < p.c.dim ? *reinterpret_cast<const uint32_t*>(q + h * p.q_head + d) : 0u;
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) m[nt][j] = -INFINITY, l[nt][j] = 0.f;
#pragma unroll
        for (int mt = 0; mt < KS; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j) o[nt][mt][j] = 0.f;
      }
      fresh = false;
    }
    const int ahead = stage == 0 ? STAGES - 1 : stage - 1;  // read in the last round: free again
    if constexpr (TMA) {
      if (lane == 0) tma.issue(p, &mk, &mv, ring + ahead * Tile::kStageBytes, bar + ahead);
      if (!mbar_wait_warp(bar + stage, parity, &abort_flag)) {
        // let this warp's copies land before the CTA's memory goes
        const int flying = min(STAGES, s.count - i);
        for (int j = 0; j < flying; ++j) {
          mbar_drain(bar + stage, parity);
          if (++stage == STAGES) stage = 0, parity ^= 1;
        }
        break;  // to the CTA's barrier, with the status raised
      }
    } else {
      cp_async_wait<STAGES - 2>();
      __syncwarp();
      copy.issue(p, ring + ahead * Tile::kStageBytes);
    }
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
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if constexpr (Cfg::kQShared) {
          uint32_t b[4];  // two matrices, named by both halves of the warp
          const int h = nt * 8 + (lane & 7);
          ldsm_x4(sq + h * (DP * 2) + (((2 * ks + ((lane >> 3) & 1)) ^ (h & 7)) << 4), b);
          mma_16816<BF16>(sc[nt][ks & 1], a, b[0], b[1]);
        } else {
          mma_16816<BF16>(sc[nt][ks & 1], a, qf[nt][ks][0], qf[nt][ks][1]);
        }
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
        x[j] = exp2_fast(x[j] - top);
        x[j + 2] = exp2_fast(x[j + 2] - top);
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

    const bool done = at.tile + 1 == at.r.t1;
    if (done || i + 1 == s.count) {
      __syncwarp();  // the ring may take the sums
      const AttnPlace to = attn_place<Cfg::kWarps, Cfg::kHeads, DP>(p, s, board, reinterpret_cast<float*>(mine), at, i,
                                                                    begun, done);
      const int h0 = at.blk * p.block_heads, nh = min(p.block_heads, p.group - h0);
      const int64_t head0 = ((int64_t)at.row * p.c.kv_heads + at.kv) * p.group + h0;
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
          if (!to.whole && lane < 4) board.ml[warp][to.slot][h] = make_float2(m[nt][j], sum);
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
    at.next(p);
    __syncwarp();
  }
  attn_merge<T, Cfg::kWarps, Cfg::kHeads, DP>(p, board, rings, Cfg::kWarpBytes);
}

// Joins the parts of the items that several CTAs share.  CTA (c, y): heads y,
// y + gridDim.y, ... of the item that begins in CTA c of the attention grid and
// goes on in the next ones, if there is one; its warps take the parts in turn.
constexpr int kJoinWarps = 8;
template <typename T>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const AttnParams p) {
  __shared__ float4 s_o[kJoinWarps][64];
  __shared__ float2 s_ml[kJoinWarps];
  griddep_wait();
  griddep_launch();
  const int4 item = p.desc[blockIdx.x];
  if (item.w == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = p.c.dim;
  const int h0 = item.z * p.block_heads, nh = min(p.block_heads, p.group - h0);
  for (int h = blockIdx.y; h < nh; h += gridDim.y) {
    AttnSum a, b;  // elements 4 lane .. and 128 + 4 lane ..
    a.clear(), b.clear();
#pragma unroll 2
    for (int i = warp; i < item.w; i += kJoinWarps) {
      const int64_t part = ((blockIdx.x + i) * 2ll + (i == 0 ? 1 : 0)) * p.block_heads + h;
      const float2 ml = p.cta_ml[part];
      const float* o = p.cta_o + part * dim;
      a.add(ml.x, ml.y, lane * 4 < dim ? *reinterpret_cast<const float4*>(o + lane * 4) : make_float4(0, 0, 0, 0));
      if (dim > 128)
        b.add(ml.x, ml.y, 128 + lane * 4 < dim ? *reinterpret_cast<const float4*>(o + 128 + lane * 4) : make_float4(0, 0, 0, 0));
    }
    __syncthreads();  // the head before has been read
    s_o[warp][lane] = make_float4(a.o[0], a.o[1], a.o[2], a.o[3]);
    if (dim > 128) s_o[warp][32 + lane] = make_float4(b.o[0], b.o[1], b.o[2], b.o[3]);
    if (lane == 0) s_ml[warp] = make_float2(a.m, a.l);
    __syncthreads();
    const int e = threadIdx.x;  // four elements
    if (e * 4 < dim) {
      AttnSum sum;
      sum.clear();
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) sum.add(s_ml[w].x, s_ml[w].y, s_o[w][e]);
      sum.put((T*)p.out + (((int64_t)item.x * p.c.kv_heads + item.y) * p.group + h0 + h) * dim + e * 4);
    }
  }
}

}  // namespace plora
