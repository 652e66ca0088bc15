// The 4-bit key/value cache: storing rows of a QKV projection into it, reading rows back, and decode attention over it.
// Each row of 64 dimensions keeps its least value (exact in BF16) and a BF16 scale, so a position costs 72 bytes per
// head and 64 dimensions for key and value together, against 256 in BF16.
#include <cuda.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "decode_math.cuh"
#include "host.hpp"
#include "kv_q4.cuh"

namespace tempo {
namespace {

constexpr uint32_t kStoreThreads = 256;

// Eight lanes take one row of 64 dimensions (a key or value of one position, head and group), 8 dimensions each: the
// least and greatest value by shuffles, scale = bf16((greatest - least) / 15), code = rne((x - least) / scale). The
// subtraction, the two divisions and the roundings are the IEEE ones, so the codes are a function of the row alone.
// A row whose scale rounds to zero (all values equal) has codes 0; one with a NaN or an infinity has a scale that is
// not finite, and reads back as NaN.
__global__ void __launch_bounds__(kStoreThreads) kv_store_q4_kernel(const uint16_t* __restrict__ rows_kv, uint32_t ld,
                                                                    uint8_t* __restrict__ cache,
                                                                    const int32_t* __restrict__ seq_of,
                                                                    const int32_t* __restrict__ pos_of, uint64_t units,
                                                                    uint32_t seqs, uint32_t kv_heads, uint32_t groups,
                                                                    uint32_t tiles) {
  pdl_wait();
  pdl_launch_dependents();
  const uint64_t unit = (uint64_t(blockIdx.x) * kStoreThreads + threadIdx.x) >> 3;
  const uint32_t li = threadIdx.x & 7u;
  if (unit >= units) return;  // whole groups of eight lanes leave together
  const uint32_t mask = 0xFFu << (threadIdx.x & 24u);
  const uint32_t per_row = 2 * kv_heads * groups;
  const uint32_t row = uint32_t(unit / per_row), column = uint32_t(unit % per_row);
  const uint32_t seq = uint32_t(seq_of[row]), pos = uint32_t(pos_of[row]);
  if (seq >= seqs || pos >= tiles * kQ4Tile) return;
  const uint32_t value = column / (kv_heads * groups), head = column / groups % kv_heads, group = column % groups;
  float x[8];
  unpack8(*reinterpret_cast<const uint4*>(rows_kv + size_t(row) * ld + column * kQ4Group + li * 8), x);
  float low = x[0], high = x[0];
  bool finite = true;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    low = fminf(low, x[j]);
    high = fmaxf(high, x[j]);
    finite = finite && fabsf(x[j]) < INFINITY;  // false for NaN too
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    low = fminf(low, __shfl_xor_sync(mask, low, o));
    high = fmaxf(high, __shfl_xor_sync(mask, high, o));
  }
  finite = (__ballot_sync(mask, finite) & mask) == mask;
  const float scale = finite ? round_bf16(__fdiv_rn(high - low, 15.f)) : __int_as_float(0x7FC00000);
  uint32_t word = 0;
  if (scale > 0.f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float code = fminf(fmaxf(rintf(__fdiv_rn(x[j] - low, scale)), 0.f), 15.f);
      word |= uint32_t(code) << (4 * j);
    }
  }
  uint8_t* block = cache + q4_block(seq, head, pos, group, kv_heads, tiles, groups);
  const uint32_t slot = pos % kQ4Tile;
  reinterpret_cast<uint32_t*>(block + value * kQ4Codes + slot * 32)[li] = word;
  if (li == 0)
    reinterpret_cast<uint32_t*>(block + 2 * kQ4Codes)[slot * 2 + value] = pack_bf16x2(scale, finite ? low : 0.f);
}

// The rows' keys and values back as BF16: code x scale + low in FP32, rounded once.
__global__ void __launch_bounds__(kStoreThreads) kv_load_q4_kernel(const uint8_t* __restrict__ cache,
                                                                   uint16_t* __restrict__ out, uint32_t ldo,
                                                                   const int32_t* __restrict__ seq_of,
                                                                   const int32_t* __restrict__ pos_of, uint64_t units,
                                                                   uint32_t seqs, uint32_t kv_heads, uint32_t groups,
                                                                   uint32_t tiles) {
  pdl_wait();
  pdl_launch_dependents();
  const uint64_t unit = (uint64_t(blockIdx.x) * kStoreThreads + threadIdx.x) >> 3;
  const uint32_t li = threadIdx.x & 7u;
  if (unit >= units) return;
  const uint32_t per_row = 2 * kv_heads * groups;
  const uint32_t row = uint32_t(unit / per_row), column = uint32_t(unit % per_row);
  const uint32_t seq = uint32_t(seq_of[row]), pos = uint32_t(pos_of[row]);
  uint4* dst = reinterpret_cast<uint4*>(out + size_t(row) * ldo + column * kQ4Group + li * 8);
  if (seq >= seqs || pos >= tiles * kQ4Tile) {
    *dst = make_uint4(0, 0, 0, 0);
    return;
  }
  const uint32_t value = column / (kv_heads * groups), head = column / groups % kv_heads, group = column % groups;
  const uint8_t* block = cache + q4_block(seq, head, pos, group, kv_heads, tiles, groups);
  const uint32_t slot = pos % kQ4Tile;
  const uint32_t word = reinterpret_cast<const uint32_t*>(block + value * kQ4Codes + slot * 32)[li];
  const uint32_t meta = reinterpret_cast<const uint32_t*>(block + 2 * kQ4Codes)[slot * 2 + value];
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = fmaf(float((word >> (4 * j)) & 15u), bf16_lo(meta), bf16_hi(meta));
  *dst = pack8(x);
}

// One CTA per (query head, sequence), four warps; eight lanes per key, 8 dimensions of each group per lane, an online
// softmax per lane group, merged over lane groups and warps at the end.
template <int G>
__global__ void __launch_bounds__(128) decode_attention_q4_kernel(const uint16_t* __restrict__ q_rows, uint32_t ldq,
                                                                  const uint8_t* __restrict__ cache,
                                                                  const int32_t* __restrict__ lengths,
                                                                  int32_t length_offset, uint16_t* __restrict__ out,
                                                                  uint32_t heads, uint32_t kv_heads, uint32_t tiles) {
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t h = blockIdx.x, s = blockIdx.y, warp = warp_id(), lane = lane_id();
  const uint32_t g = lane >> 3, li = lane & 7u, kvh = h / (heads / kv_heads);
  const int64_t want = int64_t(lengths[s]) + length_offset;
  const uint32_t capacity = tiles * kQ4Tile;
  const uint32_t len = want <= 0 ? 0u : want < int64_t(capacity) ? uint32_t(want) : capacity;
  float q[G][8], acc[G][8], qsum[G], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    load8(*reinterpret_cast<const uint4*>(q_rows + size_t(s) * ldq + h * (64 * G) + i * 64 + li * 8), q[i]);
    qsum[i] = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      q[i][d] *= kDecodeLog2e;
      qsum[i] += q[i][d];
      acc[i][d] = 0.f;
    }
  }
  for (uint32_t base = warp * 4; base < len; base += 16) {
    const uint32_t key = base + g;
    float score = 0.f;
    uint32_t vw[G], vm[G];
    if (key < len) {
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const uint8_t* block = cache + q4_block(s, kvh, key, i, kv_heads, tiles, G);
        const uint32_t slot = key % kQ4Tile;
        const uint32_t kw = reinterpret_cast<const uint32_t*>(block + slot * 32)[li];
        vw[i] = reinterpret_cast<const uint32_t*>(block + kQ4Codes + slot * 32)[li];
        const uint2 meta = reinterpret_cast<const uint2*>(block + 2 * kQ4Codes)[slot];
        vm[i] = meta.y;
        float dot = 0.f;
#pragma unroll
        for (int d = 0; d < 8; ++d) dot = fmaf(q[i][d], float((kw >> (4 * d)) & 15u), dot);
        score = fmaf(dot, bf16_lo(meta.x), fmaf(qsum[i], bf16_hi(meta.x), score));
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) score += __shfl_xor_sync(0xFFFFFFFFu, score, o);
    if (key < len) {
      const float m_new = fmaxf(m, score), c = fast_exp2(m - m_new), p = fast_exp2(score - m_new);
      m = m_new;
      l = l * c + p;
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          const float v = fmaf(float((vw[i] >> (4 * d)) & 15u), bf16_lo(vm[i]), bf16_hi(vm[i]));
          acc[i][d] = fmaf(p, v, acc[i][d] * c);
        }
    }
  }
  __shared__ float sm_m[16], sm_l[16], sm_acc[16][64 * G];
  const uint32_t part = warp * 4 + g;
  if (li == 0) {
    sm_m[part] = m;
    sm_l[part] = l;
  }
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int d = 0; d < 8; ++d) sm_acc[part][i * 64 + li * 8 + d] = acc[i][d];
  __syncthreads();
  if (threadIdx.x < 64 * G) {
    float mm = -INFINITY, ll = 0.f, aa = 0.f;
    for (int w = 0; w < 16; ++w)
      if (sm_l[w] != 0.f) mm = fmaxf(mm, sm_m[w]);
    for (int w = 0; w < 16; ++w) {
      if (sm_l[w] == 0.f) continue;
      const float f = fast_exp2(sm_m[w] - mm);
      ll = fmaf(sm_l[w], f, ll);
      aa = fmaf(sm_acc[w][threadIdx.x], f, aa);
    }
    out[size_t(s) * heads * (64 * G) + h * (64 * G) + threadIdx.x] = float_to_bf16(len == 0 ? 0.f : aa / ll);
  }
}

// What the three entry points check alike; `what` names the call.
tempo_status check_cache(const char* what, const void* cache, uint32_t seqs, uint32_t kv_heads, uint32_t head,
                         uint32_t capacity) {
  if (seqs == 0 || kv_heads == 0 || capacity == 0 || capacity % kQ4Tile || (head != 64 && head != 128))
    return fail(TEMPO_ERR_VALUE, "%s: seqs %u kv_heads %u head %u (64 or 128) capacity %u (a multiple of 16)", what,
                seqs, kv_heads, head, capacity);
  if (cache == nullptr || !aligned16(cache)) return fail(TEMPO_ERR_VALUE, "%s: the cache must be 16-byte aligned", what);
  return TEMPO_OK;
}

}  // namespace
}  // namespace tempo

using namespace tempo;

extern "C" tempo_status tempo_kv_store_q4(const void* qkv, uint32_t ldq, void* cache, const int32_t* seq_of,
                                          const int32_t* pos_of, uint32_t rows, uint32_t seqs, uint32_t heads,
                                          uint32_t kv_heads, uint32_t head, uint32_t capacity, void* stream) {
  tempo_status status = check_cache("tempo_kv_store_q4", cache, seqs, kv_heads, head, capacity);
  if (status != TEMPO_OK) return status;
  const uint64_t width = (uint64_t(heads) + 2ull * kv_heads) * head;
  if (rows == 0 || width > ldq || ldq % 8)
    return fail(TEMPO_ERR_VALUE, "tempo_kv_store_q4: rows %u, row stride %u (a multiple of 8, at least %llu)", rows, ldq,
                static_cast<unsigned long long>(width));
  if (qkv == nullptr || !aligned16(qkv) || seq_of == nullptr || pos_of == nullptr)
    return fail(TEMPO_ERR_VALUE, "tempo_kv_store_q4: 16-byte aligned rows, a sequence and a position of each are needed");
  const uint64_t units = uint64_t(rows) * 2 * kv_heads * (head / kQ4Group);
  const uint64_t blocks = (units * 8 + kStoreThreads - 1) / kStoreThreads;
  if (blocks > 0x7FFFFFFFull) return fail(TEMPO_ERR_VALUE, "tempo_kv_store_q4: %u rows are too many for one call", rows);
  return launch(kv_store_q4_kernel, dim3(uint32_t(blocks)), dim3(kStoreThreads), 0, static_cast<cudaStream_t>(stream),
                1, "kv_store_q4_kernel", static_cast<const uint16_t*>(qkv) + size_t(heads) * head, ldq,
                static_cast<uint8_t*>(cache), seq_of, pos_of, units, seqs, kv_heads, head / kQ4Group,
                capacity / kQ4Tile);
}

extern "C" tempo_status tempo_kv_load_q4(const void* cache, void* kv, uint32_t ldo, const int32_t* seq_of,
                                         const int32_t* pos_of, uint32_t rows, uint32_t seqs, uint32_t kv_heads,
                                         uint32_t head, uint32_t capacity, void* stream) {
  tempo_status status = check_cache("tempo_kv_load_q4", cache, seqs, kv_heads, head, capacity);
  if (status != TEMPO_OK) return status;
  const uint64_t width = 2ull * kv_heads * head;
  if (rows == 0 || width > ldo || ldo % 8)
    return fail(TEMPO_ERR_VALUE, "tempo_kv_load_q4: rows %u, row stride %u (a multiple of 8, at least %llu)", rows, ldo,
                static_cast<unsigned long long>(width));
  if (kv == nullptr || !aligned16(kv) || seq_of == nullptr || pos_of == nullptr)
    return fail(TEMPO_ERR_VALUE, "tempo_kv_load_q4: a 16-byte aligned output, a sequence and a position of each row are "
                "needed");
  const uint64_t units = uint64_t(rows) * 2 * kv_heads * (head / kQ4Group);
  const uint64_t blocks = (units * 8 + kStoreThreads - 1) / kStoreThreads;
  if (blocks > 0x7FFFFFFFull) return fail(TEMPO_ERR_VALUE, "tempo_kv_load_q4: %u rows are too many for one call", rows);
  return launch(kv_load_q4_kernel, dim3(uint32_t(blocks)), dim3(kStoreThreads), 0, static_cast<cudaStream_t>(stream), 1,
                "kv_load_q4_kernel", static_cast<const uint8_t*>(cache), static_cast<uint16_t*>(kv), ldo, seq_of, pos_of,
                units, seqs, kv_heads, head / kQ4Group, capacity / kQ4Tile);
}

extern "C" tempo_status tempo_decode_attention_q4(const void* q, uint32_t ldq, const void* cache,
                                                  const int32_t* lengths, int32_t length_offset, void* out,
                                                  uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head,
                                                  uint32_t capacity, void* stream) {
  tempo_status status = check_cache("tempo_decode_attention_q4", cache, seqs, kv_heads, head, capacity);
  if (status != TEMPO_OK) return status;
  if (heads == 0 || heads % kv_heads || seqs > 65535 || kv_heads > 65535)
    return fail(TEMPO_ERR_VALUE, "tempo_decode_attention_q4: seqs %u (up to 65535), heads %u must be a multiple of "
                "kv_heads %u (up to 65535)", seqs, heads, kv_heads);
  if (uint64_t(heads) * head > ldq || ldq % 8)
    return fail(TEMPO_ERR_VALUE, "tempo_decode_attention_q4: the query row stride %u must be a multiple of 8 and at "
                "least %llu", ldq, static_cast<unsigned long long>(uint64_t(heads) * head));
  if (q == nullptr || !aligned16(q) || out == nullptr || !aligned16(out) || lengths == nullptr)
    return fail(TEMPO_ERR_VALUE, "tempo_decode_attention_q4: 16-byte aligned queries and output and the lengths are "
                "needed");
  auto kernel = head == 64 ? decode_attention_q4_kernel<1> : decode_attention_q4_kernel<2>;
  return launch(kernel, dim3(heads, seqs), dim3(128), 0, static_cast<cudaStream_t>(stream), 1,
                "decode_attention_q4_kernel", static_cast<const uint16_t*>(q), ldq, static_cast<const uint8_t*>(cache),
                lengths, length_offset, static_cast<uint16_t*>(out), heads, kv_heads, capacity / kQ4Tile);
}
