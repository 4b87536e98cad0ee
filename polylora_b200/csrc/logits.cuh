// Each row's own rules on its logits: penalties for tokens the row has seen,
// biases of single tokens, and a mask of allowed tokens.
//
//   x -> x > 0 ? x / r : x * r         for tokens of the row's history
//   x -> x - f * count - p             for tokens its answer (the history past
//                                      the prompt) holds count > 0 times
//   x -> x + sum of the token's biases
//   x -> -infinity                     for tokens the mask does not allow
//
// in 32 bits, rounded once.  Bound by HBM (the logits read and written once).
//
// A token without a rule keeps its bits, or becomes -infinity, and few tokens have
// one.  So logit_copy_kernel copies the logits, 16 bytes a lane, with -infinity
// where the mask says so; logit_find_kernel finds the tokens with rules, which
// leaves the memory idle; and the rules are applied to those tokens once the copy
// is done.  The first two run side by side.  Rows few enough for all of their
// finding CTAs to wait out the copy: the copy first, and a finding CTA applies its
// own rules; few rows, cut into small parts: it copies its part too, in one launch.
// More rows: the finding first, which leaves lists, and logit_apply_kernel after
// both.  256 x 128256 bf16 logits, 4096 tokens, 64 biases and a mask: 32 us, of which
// the copy 25 (5.3 TB/s); 47 us in one kernel whose CTAs do all three.  One row: 5.6
// us, the chain of loads and barriers of the finding.
//
// The rules are found in two readings of the row's history.  The first sets a bit
// for each of its tokens; the bits, counted, give each token's place in the list of
// those with a rule.  The second adds up a word of marks and a count at that place,
// with integer atomics, so the order of threads does not matter.  Biases of one
// token are added in the order of the list.
#pragma once

#include "paged.cuh"

namespace plora {

constexpr int kRulesThreads = 256;
constexpr int kRulesStrip = 128;        // 16-byte chunks that a copying warp takes at a time
constexpr int kRulesBesideCtas = 148;  // finding CTAs that run beside the copy
constexpr int kRulesMostPart = 1 << 18; // vocabulary entries of a CTA that finds rules
// Few rows are cut into parts of no less: a CTA's tables are zeroed and counted in one
// go.  Uncut and cut, copied beside: 1 x 128256 bf16 5.6 and 4.8 us, 33 x 50257 fp32 8.3
// and 7.2.
constexpr int kRulesLeastPart = 1 << 14;
constexpr int kRulesMostSmem = 100 * 1024;
constexpr int kRulesMaxBiases = 4096;   // entries of a row's bias list
constexpr int kRulesHeld = 8;           // history entries that a thread reads at once, and of the first keeps

// Shared memory of a CTA that finds rules: bits of its part's tokens and the rank
// of each word of them; for each token with a rule its marks, itself and the first
// entry of the bias list that names it; the bias list and whether others name an
// entry's token.
__host__ __device__ constexpr int rules_words(int part) { return (part + 127) / 128 * 4; }
__host__ __device__ constexpr int rules_ruled(int part, int64_t entries) {
  return ((entries < part ? (int)entries : part) + 3) & ~3;
}
__host__ __device__ constexpr int rules_smem_bytes(int part, int64_t entries, int biases) {
  return rules_words(part) * 8 + rules_ruled(part, entries) * 12 + ((biases + 3) & ~3) * 9;
}

constexpr uint32_t kRulesSeen = 0x80000000u;   // the token is in the history
constexpr uint32_t kRulesCount = 0x7fffffffu;  // times in the answer
constexpr uint32_t kRulesNone = 0xffffffffu;   // no entry of the bias list

struct RulesParams {
  const void* x;
  void* y;
  int64_t x_row, y_row;  // elements between rows
  int64_t vocab;
  const void *tokens, *bias_tokens;  // (rows, history), (rows, biases)
  int64_t token_row, bias_row, value_row, mask_row;
  const int32_t *token_lens, *prompt_lens;  // null: the whole list; 0
  const float *repetition, *presence, *frequency, *bias_values;
  const uint32_t* allowed;
  int32_t history, biases;
  int32_t part;        // vocabulary entries of a CTA that finds rules
  bool beside;         // the finding is launched after the copy, and beside it
  bool copies;         // a finding CTA copies its part itself
  // lists (null: a finding CTA applies its rules): entries of each (row, part) and how many
  struct RulesEntry* list;
  int32_t* listed;
};

struct RulesEntry {
  int32_t token;  // offset in the part
  uint32_t mark;
  float bias;
};

// Bits i .. of a mask as the low bits of a word (a lane's chunk has at most 8).
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* m, int64_t i, int n) {
  const int s = (int)(i & 31);
  uint32_t w = m[i >> 5] >> s;
  if (s + n > 32) w |= m[(i >> 5) + 1] << (32 - s);
  return w;
}

// A 16-byte chunk with -infinity for the elements whose bit of `keep` is 0.
template <typename T>
__device__ __forceinline__ uint4 rules_masked(const uint4& u, uint32_t keep) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      if (!((keep >> i) & 1)) w[i] = 0xff800000u;
    } else {
      constexpr uint32_t kInf = std::is_same_v<T, __half> ? 0xfc00u : 0xff80u;
      if (!((keep >> (2 * i)) & 1)) w[i] = (w[i] & 0xffff0000u) | kInf;
      if (!((keep >> (2 * i + 1)) & 1)) w[i] = (w[i] & 0xffffu) | (kInf << 16);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// One token's rules.
struct RulesRow {
  float rep, pres, freq;
  __device__ __forceinline__ void read(const RulesParams& p, int64_t row) {
    rep = p.repetition ? p.repetition[row] : 1.f;
    pres = p.presence ? p.presence[row] : 0.f;
    freq = p.frequency ? p.frequency[row] : 0.f;
  }
  __device__ __forceinline__ float apply(float v, uint32_t mark) const {
    if (mark & kRulesSeen) v = v > 0.f ? v / rep : v * rep;
    const uint32_t n = mark & kRulesCount;
    return n ? v - freq * (float)n - pres : v;
  }
};

// y = x with -infinity where the mask does not allow, for strip `strip` of `count`
// elements of a row (from an element that a word of the mask begins with).  A warp
// takes a strip, counted from the first 16-byte boundary on, and a lane 16-byte
// chunks lane, lane + 32, ... of it, all four of them on their way.
template <typename T>
__device__ __forceinline__ void rules_copy(const T* x, T* y, const uint32_t* mask, int count, int strip, int lane) {
  constexpr int N = Chunk<T>::N, ROUNDS = kRulesStrip / 32;
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int head = min(count, off ? N - off : 0), first = head + strip * kRulesStrip * N;
  if (first >= count && strip != 0) return;
  auto one = [&](int i) { y[i] = mask && !(mask_bits(mask, i, 1) & 1) ? Chunk<T>::put(-INFINITY) : x[i]; };
  if ((reinterpret_cast<uintptr_t>(x) & 15) == (reinterpret_cast<uintptr_t>(y) & 15)) {
    const int chunks = (count - first) / N;  // from here on
    const uint4* from = reinterpret_cast<const uint4*>(x + first);
    uint4* to = reinterpret_cast<uint4*>(y + first);
    uint4 u[ROUNDS];
#pragma unroll
    for (int v = 0; v < ROUNDS; ++v)
      if (lane + v * 32 < chunks) u[v] = from[lane + v * 32];
    if (mask) {
      const int i0 = first + lane * N, shift = i0 & 31;  // of the chunk's mask bits in their word, in every round
      const uint32_t* m = mask + (i0 >> 5);
      uint32_t w[ROUNDS];
#pragma unroll
      for (int v = 0; v < ROUNDS; ++v) w[v] = lane + v * 32 < chunks ? m[v * N] : 0u;
#pragma unroll
      for (int v = 0; v < ROUNDS; ++v) {
        uint32_t keep = w[v] >> shift;
        if (shift + N > 32 && lane + v * 32 < chunks) keep |= m[v * N + 1] << (32 - shift);  // the rest is in the next word
        u[v] = rules_masked<T>(u[v], keep);
      }
    }
#pragma unroll
    for (int v = 0; v < ROUNDS; ++v)
      if (lane + v * 32 < chunks) to[lane + v * 32] = u[v];
    // single elements before the first chunk and after the last
    if (strip == 0 && lane < head) one(lane);
    const int tail = first + chunks * N;
    if (chunks <= kRulesStrip && tail + lane < count) one(tail + lane);
  } else {
    const int last = min(first + kRulesStrip * N, count);
#pragma unroll 8
    for (int i = (strip == 0 ? 0 : first) + lane; i < last; i += 32) one(i);
  }
}

template <typename T>
__global__ void __launch_bounds__(kRulesThreads) logit_copy_kernel(const RulesParams p) {
  const int64_t row = blockIdx.y;
  // After the finding kernel nothing need be waited for at first: it lets this one
  // start when all of its CTAs have waited for what came before.
  if (p.beside) griddep_wait();
  griddep_launch();
  rules_copy<T>((const T*)p.x + row * p.x_row, (T*)p.y + row * p.y_row,
                p.allowed ? p.allowed + row * p.mask_row : nullptr, (int)p.vocab,
                blockIdx.x * (kRulesThreads / 32) + (threadIdx.x >> 5), threadIdx.x & 31);
  // this grid's end has to mean the finding kernel's end too, for the kernel that applies its lists
  if (!p.beside && blockIdx.x + 1 == gridDim.x && blockIdx.y + 1 == gridDim.y) griddep_wait();
}

template <typename T, typename I>
__global__ void __launch_bounds__(kRulesThreads) logit_find_kernel(const RulesParams p) {
  extern __shared__ __align__(16) unsigned char rules_smem[];
  const int words = rules_words(p.part), ruled = rules_ruled(p.part, (int64_t)p.history + p.biases);
  const int entries = (p.biases + 3) & ~3;
  uint32_t* touched = reinterpret_cast<uint32_t*>(rules_smem);    // [words]
  uint32_t* rank = touched + words;                               // [words]: bits set before the word
  uint32_t* mark = rank + words;                                  // [ruled]
  int32_t* token_of = reinterpret_cast<int32_t*>(mark + ruled);   // [ruled]: offset in the part
  uint32_t* bias_of = reinterpret_cast<uint32_t*>(token_of + ruled);  // [ruled]: first entry of the token
  int32_t* bias_at = reinterpret_cast<int32_t*>(bias_of + ruled);     // [biases]: offset in the part, or -1
  float* bias_v = reinterpret_cast<float*>(bias_at + entries);        // [biases]
  uint8_t* twice = reinterpret_cast<uint8_t*>(bias_v + entries);      // [biases]: others name its token
  __shared__ int s_warp[kRulesThreads / 32];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, c0 = (int64_t)blockIdx.x * p.part;
  const int nc = (int)min((int64_t)p.part, p.vocab - c0);
  for (int i = tid; i < words; i += kRulesThreads) touched[i] = 0;
  for (int j = tid; j < entries; j += kRulesThreads) twice[j] = 0;
  // Beside the copy everything but the logits may be read at once: it lets this
  // kernel start when all of its CTAs have waited for what came before.
  if (!p.beside) {
    griddep_wait();
    griddep_launch();
  }
  const I* tok = (const I*)p.tokens + row * p.token_row;
  const I* bt = (const I*)p.bias_tokens + row * p.bias_row;
  const float* bv = p.bias_values + row * p.value_row;
  int len = 0, prompt = 0;
  if (p.history > 0) {
    len = min(p.token_lens ? p.token_lens[row] : p.history, p.history);
    if (p.prompt_lens) prompt = p.prompt_lens[row];
  }
  I bias_id = -1;
  float bias_value = 0.f;
  if (tid < p.biases) bias_id = bt[tid], bias_value = bv[tid];

  auto offset = [&](int64_t id) {  // in the part, -1: not of it
    const int64_t t = id - c0;
    return t >= 0 && t < nc ? (int)t : -1;
  };
  auto touch = [&](int at) {
    if (at >= 0) atomicOr(touched + (at >> 5), 1u << (at & 31));
  };
  auto slot = [&](int at) { return rank[at >> 5] + __popc(touched[at >> 5] & ((1u << (at & 31)) - 1)); };
  // kRulesHeld entries of a thread at a time, loaded before any is looked at
  auto read = [&](int i0, int (&at)[kRulesHeld]) {
    I id[kRulesHeld];
#pragma unroll
    for (int k = 0; k < kRulesHeld; ++k) id[k] = tok[min(i0 + k * kRulesThreads, len - 1)];
#pragma unroll
    for (int k = 0; k < kRulesHeld; ++k) at[k] = i0 + k * kRulesThreads < len ? offset(id[k]) : -1;
  };
  constexpr int kRound = kRulesHeld * kRulesThreads;
  int held[kRulesHeld];  // the first round's, kept for the second reading
#pragma unroll
  for (int k = 0; k < kRulesHeld; ++k) held[k] = -1;
  if (len > 0) read(tid, held);
  if (p.copies) {  // the barriers up to the applying order it and the copy
    const uint32_t* mask = p.allowed ? p.allowed + row * p.mask_row + c0 / 32 : nullptr;
    for (int strip = tid / 32; strip * kRulesStrip * Chunk<T>::N < nc; strip += kRulesThreads / 32)
      rules_copy<T>((const T*)p.x + row * p.x_row + c0, (T*)p.y + row * p.y_row + c0, mask, nc, strip, tid & 31);
  }
  __syncthreads();  // the bits are zero
#pragma unroll
  for (int k = 0; k < kRulesHeld; ++k) touch(held[k]);
  for (int i0 = tid + kRound; i0 < len; i0 += kRound) {
    int at[kRulesHeld];
    read(i0, at);
#pragma unroll
    for (int k = 0; k < kRulesHeld; ++k) touch(at[k]);
  }
  for (int j = tid; j < entries; j += kRulesThreads) {
    if (j != tid) bias_id = j < p.biases ? bt[j] : -1, bias_value = j < p.biases ? bv[j] : 0.f;
    const int at = offset(bias_id);
    bias_at[j] = at;
    bias_v[j] = bias_value;
    touch(at);
  }
  __syncthreads();
  int total;
  {  // ranks: a thread takes every 256th four words of neighbouring ones
    int before = 0;  // of the rounds before
    for (int w0 = 0; w0 < words; w0 += 4 * kRulesThreads) {
      const int w = w0 + 4 * tid;
      uint4 b = make_uint4(0, 0, 0, 0);
      if (w < words) b = *reinterpret_cast<const uint4*>(touched + w);
      const int n0 = __popc(b.x), n1 = n0 + __popc(b.y), n2 = n1 + __popc(b.z), n3 = n2 + __popc(b.w);
      const int at = before + block_scan<kRulesThreads / 32>(n3, s_warp, &total);
      if (w < words) *reinterpret_cast<uint4*>(rank + w) = make_uint4(at, at + n0, at + n1, at + n2);
      before += total;
    }
    total = before;
    for (int r = tid; r < total; r += kRulesThreads) mark[r] = 0, bias_of[r] = kRulesNone;
  }
  __syncthreads();
  auto count = [&](int at, int i) {
    if (at < 0) return;
    const int r = slot(at);
    token_of[r] = at;  // the same from each of the token's entries
    if (i >= prompt) atomicAdd(mark + r, 1u);
    atomicOr(mark + r, kRulesSeen);
  };
#pragma unroll
  for (int k = 0; k < kRulesHeld; ++k) count(held[k], tid + k * kRulesThreads);
  for (int i0 = tid + kRound; i0 < len; i0 += kRound) {
    int at[kRulesHeld];
    read(i0, at);
#pragma unroll
    for (int k = 0; k < kRulesHeld; ++k) count(at[k], i0 + k * kRulesThreads);
  }
  for (int j = tid; j < p.biases; j += kRulesThreads) {
    const int at = bias_at[j];
    if (at < 0) continue;
    const int r = slot(at);
    token_of[r] = at;
    atomicMin(bias_of + r, (uint32_t)j);
  }
  RulesRow rules;
  if (!p.list) rules.read(p, row);
  __syncthreads();
  if (p.biases > 0) {
    for (int j = tid; j < p.biases; j += kRulesThreads) {
      if (bias_at[j] < 0) continue;
      const uint32_t first = bias_of[slot(bias_at[j])];
      if (first != j) twice[first] = 1;
    }
    __syncthreads();
    // A warp adds up a token's biases, looking at 32 entries at a time; one by one, a
    // token named twice among 300 took 8 us.
    const int lane = tid & 31;
    for (int j0 = tid - lane; j0 < p.biases; j0 += kRulesThreads) {
      uint32_t todo = __ballot_sync(0xffffffffu, j0 + lane < p.biases && twice[j0 + lane]);
      for (; todo; todo &= todo - 1) {
        const int j = j0 + __ffs(todo) - 1, token = bias_at[j];
        float sum = bias_v[j];
#pragma unroll 4
        for (int o0 = j0; o0 < p.biases; o0 += 32) {
          const int o = o0 + lane;
          uint32_t same = __ballot_sync(0xffffffffu, o > j && o < p.biases && bias_at[o] == token);
          for (; same; same &= same - 1) sum += bias_v[o0 + __ffs(same) - 1];
        }
        if (lane == 0) bias_v[j] = sum;  // read by this warp alone until the barrier
      }
    }
    __syncthreads();
  }
  auto bias = [&](int r) { return bias_of[r] == kRulesNone ? 0.f : bias_v[bias_of[r]]; };

  if (p.list) {
    const int64_t at = row * gridDim.x + blockIdx.x;
    RulesEntry* list = p.list + at * ruled;
    for (int r = tid; r < total; r += kRulesThreads) list[r] = RulesEntry{token_of[r], mark[r], bias(r)};
    if (tid == 0) p.listed[at] = total;
    return;
  }
  if (p.beside) {
    griddep_wait();
    griddep_launch();
  }
  const uint32_t* mask = p.allowed ? p.allowed + row * p.mask_row : nullptr;
  const T* x = (const T*)p.x + row * p.x_row;
  T* y = (T*)p.y + row * p.y_row;
  for (int r0 = tid; r0 < total; r0 += 4 * kRulesThreads) {
    int64_t i[4];
    T v[4];
    uint32_t allowed[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // loads first, past the end of the last one
      i[k] = c0 + token_of[min(r0 + k * kRulesThreads, total - 1)];
      v[k] = x[i[k]];  // in place: still the logit, or -infinity behind the mask
      allowed[k] = mask ? mask[i[k] >> 5] >> (i[k] & 31) : 1u;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = r0 + k * kRulesThreads;
      if (r < total && (allowed[k] & 1)) y[i[k]] = Chunk<T>::put(rules.apply(Chunk<T>::get(v[k]), mark[r]) + bias(r));
    }
  }
}

// Applies the lists: CTA (x, row) every gridDim.x-th 256 entries of the row's.
template <typename T>
__global__ void __launch_bounds__(kRulesThreads) logit_apply_kernel(const RulesParams p) {
  const int64_t row = blockIdx.y;
  const int parts = (int)((p.vocab + p.part - 1) / p.part), ruled = rules_ruled(p.part, (int64_t)p.history + p.biases);
  const uint32_t* mask = p.allowed ? p.allowed + row * p.mask_row : nullptr;
  const T* x = (const T*)p.x + row * p.x_row;
  T* y = (T*)p.y + row * p.y_row;
  griddep_wait();
  griddep_launch();
  RulesRow rules;
  rules.read(p, row);
  for (int part = 0; part < parts; ++part) {
    const int64_t at = row * parts + part;
    const int total = p.listed[at];
    for (int r = blockIdx.x * kRulesThreads + threadIdx.x; r < total; r += gridDim.x * kRulesThreads) {
      const RulesEntry e = p.list[at * ruled + r];
      const int64_t i = (int64_t)part * p.part + e.token;
      const T v = x[i];  // in place: still the logit, or -infinity behind the mask
      if (!mask || (mask[i >> 5] >> (i & 31) & 1)) y[i] = Chunk<T>::put(rules.apply(Chunk<T>::get(v), e.mark) + e.bias);
    }
  }
}

}  // namespace plora
