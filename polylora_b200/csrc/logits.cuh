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
// A token without a rule keeps its bits, or becomes -infinity, and few tokens have
// one.  So half of a CTA's warps copy a chunk of a row's logits, 16 bytes a lane,
// putting -infinity where the mask says so, while the other half works out the
// chunk's rules; then all of them go over the tokens with rules.
//
// The rules are found in two readings of the row's history.  The first sets a bit
// for each of the chunk's tokens; the bits, counted, give the list of those tokens
// and each one's place in it.  The second adds up a word of marks and a count at
// that place, with integer atomics, so the order of threads does not matter.  A
// bias belongs to the first entry of the list that names its token, which adds up
// the others in their order.  With a bit per token and eight bytes per token that
// has a rule a chunk can be large, and a row's history is read by few CTAs.
#pragma once

#include "paged.cuh"

namespace plora {

constexpr int kRulesThreads = 256;
constexpr int kRulesHalf = kRulesThreads / 2;  // threads that copy, threads that find the rules
constexpr int kRulesStep = 8192;               // vocabulary entries of a CTA: this many times 1, 2, 3 or 4
constexpr int kRulesMaxChunk = 4 * kRulesStep;
constexpr int kRulesMaxBiases = 4096;          // entries of a row's bias list
constexpr int kRulesHeld = 16;                 // history entries that a thread keeps between its two readings

// Shared memory of a call with a history or biases: bits and the rank of each word
// of them; for each token with a rule its marks, its place in the chunk and its
// entry of the bias list; the bias list and its sums.
__host__ __device__ constexpr int rules_ruled(int chunk, int64_t entries) {
  return ((entries < chunk ? (int)entries : chunk) + 3) & ~3;
}
__host__ __device__ constexpr int rules_smem_bytes(int chunk, int64_t entries, int biases) {
  return (chunk / 32 + 4) * 6 + rules_ruled(chunk, entries) * 8 + biases * 12;
}

constexpr uint32_t kRulesSeen = 0x80000000u;    // the token is in the history
constexpr uint32_t kRulesBiased = 0x40000000u;  // the token has a bias
constexpr uint32_t kRulesCount = 0x3fffffffu;   // times in the answer

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
  int32_t history, biases, chunk;
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

template <typename T, typename I>
__global__ void __launch_bounds__(kRulesThreads) logit_rules_kernel(const RulesParams p) {
  constexpr int N = Chunk<T>::N, VECS = 8;  // 16-byte chunks that a copying thread has on their way
  extern __shared__ __align__(16) unsigned char rules_smem[];
  const int words = p.chunk / 32, ruled = rules_ruled(p.chunk, (int64_t)p.history + p.biases);
  uint32_t* touched = reinterpret_cast<uint32_t*>(rules_smem);        // [words, four more]
  uint32_t* mark = touched + words + 4;                               // [ruled]
  int32_t* bias_at = reinterpret_cast<int32_t*>(mark + ruled);        // [biases]: place in the chunk, or -1
  float* bias_v = reinterpret_cast<float*>(bias_at + p.biases);       // [biases]
  float* bias_sum = bias_v + p.biases;                                // [biases]
  uint16_t* rank = reinterpret_cast<uint16_t*>(bias_sum + p.biases);  // [words, four more]: bits set before the word
  uint16_t* place_of = rank + words + 4;                              // [ruled]
  uint16_t* bias_of = place_of + ruled;                               // [ruled]: a biased token's entry
  __shared__ int s_warp[kRulesHalf / 32];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, c0 = (int64_t)blockIdx.x * p.chunk;
  const int nc = (int)min((int64_t)p.chunk, p.vocab - c0);
  const bool marks = p.history > 0 || p.biases > 0;
  if (marks)
    for (int i = tid; i < words + 4; i += kRulesThreads) touched[i] = 0;
  __syncthreads();
  griddep_wait();
  griddep_launch();
  const uint32_t* mask = p.allowed ? p.allowed + row * p.mask_row : nullptr;
  const T* x = (const T*)p.x + row * p.x_row + c0;
  T* y = (T*)p.y + row * p.y_row + c0;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (p.repetition) rep = p.repetition[row];
  if (p.presence) pres = p.presence[row];
  if (p.frequency) freq = p.frequency[row];

  if (tid >= kRulesHalf) {
    if (x != y || mask) {
      const int th = tid - kRulesHalf;
      // 16-byte chunks where x and y lie alike on them, single elements before and after
      const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
      const bool alike = (reinterpret_cast<uintptr_t>(x) & 15) == (reinterpret_cast<uintptr_t>(y) & 15);
      const int head = alike ? min(nc, off ? N - off : 0) : nc;
      const int vecs = (nc - head) / N;
      const bool even = head % N == 0;  // the mask bits of a 16-byte chunk lie in one word (c0 is a multiple of 32)
      for (int j0 = th; j0 < vecs; j0 += VECS * kRulesHalf) {
        uint4 u[VECS];
        uint32_t w0[VECS], w1[VECS];
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
          const int i = head + min(j0 + v * kRulesHalf, vecs - 1) * N;
          u[v] = *reinterpret_cast<const uint4*>(x + i);
          w0[v] = w1[v] = ~0u;
          if (mask) {
            w0[v] = mask[(c0 + i) >> 5];
            if (!even) w1[v] = mask[(c0 + i + N - 1) >> 5];
          }
        }
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
          const int j = j0 + v * kRulesHalf, i = head + j * N;
          if (j < vecs) *reinterpret_cast<uint4*>(y + i) = rules_masked<T>(u[v], __funnelshift_r(w0[v], w1[v], i & 31));
        }
      }
      auto one = [&](int i) { y[i] = mask && !(mask_bits(mask, c0 + i, 1) & 1) ? Chunk<T>::put(-INFINITY) : x[i]; };
#pragma unroll 4
      for (int i = th; i < head; i += kRulesHalf) one(i);
      for (int i = head + vecs * N + th; i < nc; i += kRulesHalf) one(i);
    }
  } else if (marks) {
    const I* tok = (const I*)p.tokens + row * p.token_row;
    const I* bt = (const I*)p.bias_tokens + row * p.bias_row;
    const float* bv = p.bias_values + row * p.value_row;
    const int len = p.history > 0 ? min(p.token_lens ? p.token_lens[row] : p.history, p.history) : 0;
    const int prompt = p.history > 0 && p.prompt_lens ? p.prompt_lens[row] : 0;
    auto place = [&](int64_t id) {  // -1: not of this chunk
      const int64_t t = id - c0;
      return t >= 0 && t < nc ? (int)t : -1;
    };
    auto touch = [&](int t) {
      if (t >= 0) atomicOr(touched + (t >> 5), 1u << (t & 31));
    };
    auto slot = [&](int t) { return rank[t >> 5] + __popc(touched[t >> 5] & ((1u << (t & 31)) - 1)); };
    for (int j = tid; j < p.biases; j += kRulesHalf) {
      const int t = place(bt[j]);
      bias_at[j] = t;
      bias_v[j] = bv[j];
      touch(t);
    }
    int held[kRulesHeld];
#pragma unroll
    for (int k = 0; k < kRulesHeld; ++k) {
      const int i = tid + k * kRulesHalf;
      held[k] = i < len ? place(tok[i]) : -1;
    }
#pragma unroll
    for (int k = 0; k < kRulesHeld; ++k) touch(held[k]);
#pragma unroll 4
    for (int i = tid + kRulesHeld * kRulesHalf; i < len; i += kRulesHalf) touch(place(tok[i]));
    named_barrier(1, kRulesHalf);
    {  // ranks: a thread takes neighbouring words
      const int per = (words + kRulesHalf - 1) / kRulesHalf, first = min(tid * per, words), last = min(first + per, words);
      int mine = 0;
      for (int w = first; w < last; ++w) mine += __popc(touched[w]);
      int before = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, d);
        if ((tid & 31) >= d) before += v;
      }
      if ((tid & 31) == 31) s_warp[tid >> 5] = before;
      before -= mine;
      named_barrier(1, kRulesHalf);
      for (int w = 0; w < (tid >> 5); ++w) before += s_warp[w];
      for (int w = first; w < last; ++w) {
        rank[w] = (uint16_t)before;
        for (uint32_t bits = touched[w]; bits; bits &= bits - 1, ++before) {
          place_of[before] = (uint16_t)(w * 32 + __ffs(bits) - 1);
          mark[before] = 0;
        }
      }
    }
    named_barrier(1, kRulesHalf);
    auto count = [&](int t, int i) {
      if (t < 0) return;
      uint32_t* w = mark + slot(t);
      if (i >= prompt) atomicAdd(w, 1u);
      atomicOr(w, kRulesSeen);
    };
#pragma unroll
    for (int k = 0; k < kRulesHeld; ++k) count(held[k], tid + k * kRulesHalf);
#pragma unroll 4
    for (int i = tid + kRulesHeld * kRulesHalf; i < len; i += kRulesHalf) count(place(tok[i]), i);
    for (int j = tid; j < p.biases; j += kRulesHalf) {
      const int t = bias_at[j];
      if (t < 0) continue;
      bool owner = true;
      for (int k = 0; k < j && owner; ++k) owner = bias_at[k] != t;
      if (!owner) continue;
      float v = bias_v[j];
      for (int k = j + 1; k < p.biases; ++k)
        if (bias_at[k] == t) v += bias_v[k];
      bias_sum[j] = v;
      const int r = slot(t);
      bias_of[r] = (uint16_t)j;
      atomicOr(mark + r, kRulesBiased);
    }
  }
  if (!marks) return;
  __syncthreads();

  const int total = s_warp[0] + s_warp[1] + s_warp[2] + s_warp[3];
  static_assert(kRulesHalf == 128, "four warps' counts");
#pragma unroll 4
  for (int r = tid; r < total; r += kRulesThreads) {
    const int i = place_of[r];
    float v = Chunk<T>::get(x[i]);  // in place: still the logit, or -infinity behind the mask
    const uint32_t w = mark[r];
    if (w & kRulesSeen) v = v > 0.f ? v / rep : v * rep;
    const uint32_t n = w & kRulesCount;
    if (n) v = v - freq * (float)n - pres;
    if (w & kRulesBiased) v += bias_sum[bias_of[r]];
    if (!mask || (mask_bits(mask, c0 + i, 1) & 1)) y[i] = Chunk<T>::put(v);
  }
}

}  // namespace plora
