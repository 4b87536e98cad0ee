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
// A CTA takes a chunk of a row's vocabulary: it reads the row's history and
// marks the tokens that fall in its chunk in shared-memory words (integer
// atomics, so the order of threads does not matter), then passes over the
// logits once, 16 bytes a lane.  Biases of one token are added in the order of
// the list: one entry per token sums the others in.
#pragma once

#include "paged.cuh"

namespace plora {

constexpr int kRulesThreads = 256;
constexpr int kRulesChunk = 8192;     // vocabulary entries of a CTA
constexpr int kRulesMaxBiases = 4096; // entries of a row's bias list

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
  int32_t history, biases;
};

// Bits i .. of a mask as the low bits of a word (a lane's chunk has at most 8).
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* m, int64_t i, int n) {
  const int s = (int)(i & 31);
  uint32_t w = m[i >> 5] >> s;
  if (s + n > 32) w |= m[(i >> 5) + 1] << (32 - s);
  return w;
}

template <typename T, typename I>
__global__ void __launch_bounds__(kRulesThreads) logit_rules_kernel(const RulesParams p) {
  constexpr int N = Chunk<T>::N;
  extern __shared__ __align__(16) unsigned char rules_smem[];
  uint32_t* word = reinterpret_cast<uint32_t*>(rules_smem);                      // [chunk]
  uint16_t* first = reinterpret_cast<uint16_t*>(word + kRulesChunk);       // [chunk]: an entry of the token's
  float* sum = reinterpret_cast<float*>(first + kRulesChunk);              // [biases]
  uint8_t* twice = reinterpret_cast<uint8_t*>(sum + p.biases);             // [biases]: others name its token
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y, c0 = (int64_t)blockIdx.x * kRulesChunk;
  const int nc = (int)min((int64_t)kRulesChunk, p.vocab - c0);
  const bool marks = p.history > 0 || p.biases > 0;
  if (marks)
    for (int i = tid; i < kRulesChunk / 4; i += kRulesThreads) reinterpret_cast<uint4*>(word)[i] = make_uint4(0, 0, 0, 0);
  for (int i = tid; i < p.biases; i += kRulesThreads) twice[i] = 0;
  griddep_wait();
  griddep_launch();

  float rep = 1.f, pres = 0.f, freq = 0.f;
  if (marks) {
    __syncthreads();
    if (p.history > 0) {
      const I* tok = (const I*)p.tokens + row * p.token_row;
      const int len = p.token_lens ? min(max(p.token_lens[row], 0), p.history) : p.history;
      const int prompt = p.prompt_lens ? p.prompt_lens[row] : 0;
      for (int i = tid; i < len; i += kRulesThreads) {
        const int64_t t = (int64_t)tok[i] - c0;
        if (t >= 0 && t < nc) {
          // the first sighting sets the mark; answers count on
          if (i >= prompt) atomicAdd(word + t, 1u);
          atomicOr(word + t, kRulesSeen);
        }
      }
      if (p.repetition) rep = p.repetition[row];
      if (p.presence) pres = p.presence[row];
      if (p.frequency) freq = p.frequency[row];
    }
    const I* bt = (const I*)p.bias_tokens + row * p.bias_row;
    const float* bv = p.bias_values + row * p.value_row;
    if (p.biases > 0) {
      for (int j = tid; j < p.biases; j += kRulesThreads) {
        const int64_t t = (int64_t)bt[j] - c0;
        if (t >= 0 && t < nc) {
          atomicOr(word + t, kRulesBiased);
          first[t] = (uint16_t)j;  // any one of the token's entries
        }
      }
      __syncthreads();
      for (int j = tid; j < p.biases; j += kRulesThreads) {
        const int64_t t = (int64_t)bt[j] - c0;
        if (t >= 0 && t < nc && first[t] != j) twice[first[t]] = 1;
      }
      __syncthreads();
      for (int j = tid; j < p.biases; j += kRulesThreads) {
        const int64_t t = (int64_t)bt[j] - c0;
        if (t < 0 || t >= nc || first[t] != j) continue;
        float v = bv[j];
        if (twice[j]) {
          v = 0.f;
          for (int k = 0; k < p.biases; ++k)
            if ((int64_t)bt[k] - c0 == t) v += bv[k];
        }
        sum[j] = v;
      }
    }
    __syncthreads();
  }

  const uint32_t* mask = p.allowed ? p.allowed + row * p.mask_row : nullptr;
  const T* x = (const T*)p.x + row * p.x_row + c0;
  T* y = (T*)p.y + row * p.y_row + c0;
  auto rule = [&](float v, int i) {
    const uint32_t w = marks ? word[i] : 0u;
    if (w) {
      if (w & kRulesSeen) v = v > 0.f ? v / rep : v * rep;
      const uint32_t n = w & kRulesCount;
      if (n) v = v - freq * (float)n - pres;
      if (w & kRulesBiased) v += sum[first[i]];
    }
    return v;
  };
  auto one = [&](int i) {
    const float v = rule(Chunk<T>::get(x[i]), i);
    y[i] = Chunk<T>::put(mask && !(mask_bits(mask, c0 + i, 1) & 1) ? -INFINITY : v);
  };
  // 16-byte chunks where x and y lie alike on them, single elements before and after
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const bool alike = (reinterpret_cast<uintptr_t>(x) & 15) == (reinterpret_cast<uintptr_t>(y) & 15);
  const int head = alike ? min(nc, off ? N - off : 0) : nc;
  const int vecs = (nc - head) / N;
  for (int i = tid; i < head; i += kRulesThreads) one(i);
  for (int j = tid; j < vecs; j += kRulesThreads) {
    const int i = head + j * N;
    float f[N];
    Chunk<T>::load(*reinterpret_cast<const uint4*>(x + i), f);
    const uint32_t bits = mask ? mask_bits(mask, c0 + i, N) : 0xffu;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      f[e] = rule(f[e], i + e);
      if (!((bits >> e) & 1)) f[e] = -INFINITY;
    }
    *reinterpret_cast<uint4*>(y + i) = Chunk<T>::store(f);
  }
  for (int i = head + vecs * N + tid; i < nc; i += kRulesThreads) one(i);
}

}  // namespace plora
