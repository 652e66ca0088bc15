// Log probabilities of given tokens, the entropy of each row's distribution and its likeliest alternatives, from
// logits: with m the row's maximum, l = sum e^(x - m) and t = sum (x - m) e^(x - m),
//   log p(id) = x[id] - m - ln l,   entropy = ln l - t / l,
// and the alternatives are the greatest logits, ties going to the lower index.
#include <cfloat>

#include <cuda_runtime.h>

#include "common.cuh"
#include "host.hpp"

namespace tempo {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxTop = 32;
constexpr float kLog2e = 1.4426950408889634f;

struct LogprobParams {
  const void* logits;
  uint64_t ld;
  const int32_t* ids;
  uint32_t vocab, top;
  float* logprob;
  float* entropy;
  float* top_logprob;
  int32_t* top_ids;
};

template <typename T>
__device__ __forceinline__ float logit(const T* row, uint32_t i);
template <>
__device__ __forceinline__ float logit(const float* row, uint32_t i) { return row[i]; }
template <>
__device__ __forceinline__ float logit(const uint16_t* row, uint32_t i) { return bf16_to_float(row[i]); }

// A logit and its index as one unsigned key: greater logits first (NaN before all, -0 equal to +0), then the lower
// index. Keys of a row differ, so an order by key has no ties.
__device__ __forceinline__ uint64_t order_key(float x, uint32_t index) {
  const uint32_t bits = __float_as_uint(x + 0.f);
  uint32_t rank = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
  if (x != x) rank = 0xFFFFFFFFu;
  return uint64_t(rank) << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t rank = uint32_t(key >> 32);
  return __uint_as_float(rank & 0x80000000u ? rank & 0x7FFFFFFFu : ~rank);
}

__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = warp_sum(v);
  if (lane_id() == 0) scratch[warp_id()] = v;
  __syncthreads();
  float sum = 0.f;
  for (uint32_t w = 0; w < kThreads / 32; ++w) sum += scratch[w];
  __syncthreads();
  return sum;
}

// One CTA per row: the maximum, the sums, then the alternatives one by one, each the greatest key below the last.
template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(LogprobParams p) {
  __shared__ float scratch[kThreads / 32];
  __shared__ uint64_t keys[kThreads / 32];
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t r = blockIdx.x;
  const T* row = static_cast<const T*>(p.logits) + size_t(r) * p.ld;
  float m = -INFINITY;
  for (uint32_t i = threadIdx.x; i < p.vocab; i += kThreads) m = fmaxf(m, logit(row, i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  if (lane_id() == 0) scratch[warp_id()] = m;
  __syncthreads();
  for (uint32_t w = 0; w < kThreads / 32; ++w) m = fmaxf(m, scratch[w]);
  __syncthreads();
  const float base = fmaxf(m, -FLT_MAX);
  float l = 0.f, t = 0.f;
  for (uint32_t i = threadIdx.x; i < p.vocab; i += kThreads) {
    const float d = logit(row, i) - base, e = fast_exp2(d * kLog2e);
    l += e;
    t = fmaf(fmaxf(d, -1000.f), e, t);
  }
  l = block_sum(l, scratch);
  t = block_sum(t, scratch);
  const float log_l = logf(l);
  const bool empty = l == 0.f;
  if (threadIdx.x == 0) {
    const uint32_t id = uint32_t(p.ids[r]);
    p.logprob[r] = id >= p.vocab ? 0.f : empty ? -INFINITY : logit(row, id) - base - log_l;
    p.entropy[r] = empty ? 0.f : log_l - t / l;
  }
  uint64_t last = ~0ull;
  for (uint32_t k = 0; k < p.top; ++k) {
    uint64_t best = 0;
    for (uint32_t i = threadIdx.x; i < p.vocab; i += kThreads) {
      const uint64_t key = order_key(logit(row, i), i);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xFFFFFFFFu, best, o);
      best = other > best ? other : best;
    }
    if (lane_id() == 0) keys[warp_id()] = best;
    __syncthreads();
    for (uint32_t w = 0; w < kThreads / 32; ++w) best = keys[w] > best ? keys[w] : best;
    __syncthreads();
    last = best;
    if (threadIdx.x == 0) {
      p.top_ids[size_t(r) * p.top + k] = int32_t(0xFFFFFFFFu - uint32_t(best));
      p.top_logprob[size_t(r) * p.top + k] = empty ? -INFINITY : key_logit(best) - base - log_l;
    }
  }
}

}  // namespace
}  // namespace tempo

using namespace tempo;

extern "C" tempo_status tempo_token_logprobs(const void* logits, uint64_t ld, uint32_t bf16, const int32_t* ids,
                                             uint32_t rows, uint32_t vocab, uint32_t top, float* logprob,
                                             float* entropy, float* top_logprob, int32_t* top_ids, void* stream) {
  if (rows == 0 || vocab == 0 || vocab > 0x7FFFFFFFu || rows > 0x7FFFFFFFu || ld < vocab)
    return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: rows %u vocab %u, row stride %llu (at least the vocabulary)", rows,
                vocab, static_cast<unsigned long long>(ld));
  if (top > kMaxTop || top > vocab)
    return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: %u alternatives of %u tokens (at most %u)", top, vocab, kMaxTop);
  if (bf16 > 1) return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: the logits are FP32 (0) or BF16 (1), got %u", bf16);
  if (logits == nullptr || (reinterpret_cast<uintptr_t>(logits) & (bf16 ? 1u : 3u)) || ids == nullptr ||
      logprob == nullptr || entropy == nullptr || (top > 0 && (top_logprob == nullptr || top_ids == nullptr)))
    return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: aligned logits, ids and every output are needed");
  const LogprobParams p{logits, ld, ids, vocab, top, logprob, entropy, top_logprob, top_ids};
  auto kernel = bf16 ? token_logprobs_kernel<uint16_t> : token_logprobs_kernel<float>;
  return launch(kernel, dim3(rows), dim3(kThreads), 0, static_cast<cudaStream_t>(stream), 1, "token_logprobs_kernel", p);
}
