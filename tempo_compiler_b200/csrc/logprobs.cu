// Log probabilities of given tokens, the entropy of each row's distribution and its likeliest alternatives, from
// logits: with m the row's maximum, l = sum e^(x - m) and t = sum (x - m) e^(x - m),
//   log p(id) = x[id] - m - ln l,   entropy = ln l - t / l,
// and the alternatives are the greatest logits, ties going to the lower index.
//
// One pass over the logits bounds the kernel (four or two bytes a logit): each thread keeps a running maximum and the
// two sums rescaled to it, and notes the maximum of every cell (its share of a few chunks) in shared memory. The
// alternatives cost that pass nothing more. From the threads' maxima, the CTA takes the top-th greatest of its lane
// groups' as a bar, a lower bound on the top-th greatest logit that only about as many logits pass; the CTA reads again
// the few cells whose maximum does, gathers the logits at or above the bar as keys (which join a logit with its index,
// and so have no ties) and sorts them by counting. A row with more
// ties at the bar than the lists hold, or with a NaN, is searched exactly, at a slower pace. Few rows are split over the
// CTAs of a cluster, whose sums and sorted candidates the first one merges. (Collecting candidates on the way, against
// a threshold that rose with the row, took 230 us for 8192 BF16 rows of 50257 when this took 163.)

#include <cuda_runtime.h>

#include "common.cuh"
#include "host.hpp"

namespace tempo {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32;
// 16-byte words of one thread and chunk: as many as 64 registers hold (four CTAs an SM). 8192 BF16 rows with one alternative
// take 160 us with five words, 163 with four, 172 with three, 175 with six, which spill.
constexpr uint32_t kVectors = 5;
constexpr uint32_t kChunk = kThreads * kVectors;    // a chunk, in 16-byte words
constexpr uint32_t kLanes = 4;                      // of a group whose greatest keys give a threshold
constexpr uint32_t kGroups = kThreads / kLanes;
constexpr uint32_t kMaxTop = 32;
constexpr uint32_t kCapacity = 1024;                // candidates
constexpr uint32_t kThin = kCapacity - kThreads;    // the second look thins above this
constexpr uint32_t kCells = 32;                     // of a thread
constexpr uint32_t kListed = 512;                   // cells read again
constexpr uint32_t kMaxChunks = 8;                  // CTAs of a cluster sharing one row
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
static_assert(kGroups >= 2 * kMaxTop, "thinning drops at least half of the groups");

struct LogprobParams {
  const void* logits;
  uint64_t ld;
  const int32_t* ids;
  uint32_t rows, vocab, top, chunks;
  float* logprob;
  float* entropy;
  float* top_logprob;
  int32_t* top_ids;
  // With slot_of, row r's results go to row slot * rows + r of the outputs, slot = slot_of[r] + slot_offset, and nowhere
  // unless 0 <= slot < slots.
  const int32_t* slot_of;
  int32_t slot_offset;
  uint32_t slots;
};

// The least of three floats (PTX min.f32 with three inputs); a NaN operand is ignored, as by fminf.
__device__ __forceinline__ float fmin3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The logits of 32-bit words: how many, the pairs of them as floats, and the greatest and least of several words.
template <typename T>
struct Logits;
template <>
struct Logits<float> {
  static constexpr uint32_t kPerWord = 1;                 // logits of a 32-bit word
  static constexpr uint32_t kMasked = 0xFF800000u;        // a word of -infinity
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  template <uint32_t N>
  static __device__ __forceinline__ void pair(const uint32_t (&w)[N], uint32_t i, float& a, float& b) {
    a = __uint_as_float(w[2 * i]);
    b = __uint_as_float(w[2 * i + 1]);
  }
  template <uint32_t N>
  static __device__ __forceinline__ void range(const uint32_t (&w)[N], float& most, float& least) {
    most = least = __uint_as_float(w[0]);
#pragma unroll
    for (uint32_t i = 1; i < N; i += 2) {
      const float a = __uint_as_float(w[i]), b = __uint_as_float(w[i + 1 < N ? i + 1 : i]);
      most = fmax3(most, a, b);
      least = fmin3(least, a, b);
    }
  }
};
template <>
struct Logits<uint16_t> {
  static constexpr uint32_t kPerWord = 2;
  static constexpr uint32_t kMasked = 0xFF80FF80u;
  static __device__ __forceinline__ float one(const uint16_t* p) { return bf16_to_float(*p); }
  template <uint32_t N>
  static __device__ __forceinline__ void pair(const uint32_t (&w)[N], uint32_t i, float& a, float& b) {
    a = bf16_lo(w[i]);
    b = bf16_hi(w[i]);
  }
  template <uint32_t N>
  static __device__ __forceinline__ void range(const uint32_t (&w)[N], float& most, float& least) {
    uint32_t high = w[0], low = w[0];
#pragma unroll
    for (uint32_t i = 1; i < N; ++i) {
      asm("max.bf16x2 %0, %0, %1;" : "+r"(high) : "r"(w[i]));
      asm("min.bf16x2 %0, %0, %1;" : "+r"(low) : "r"(w[i]));
    }
    most = fmaxf(bf16_lo(high), bf16_hi(high));
    least = fminf(bf16_lo(low), bf16_hi(low));
  }
};

__device__ __forceinline__ uint4 ld_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// A logit and its index as one unsigned key: greater logits first (NaN before all, -0 equal to +0), then the lower
// index. Keys of a row differ, so an order by key has no ties. 0 is below every key.
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

struct Candidates {
  uint64_t keys[kCapacity];
  uint64_t group[kGroups];
  uint64_t threshold;
  uint32_t count;
  float bar;
  uint32_t cells;                       // cells whose greatest logit reaches the bar
  uint32_t cell[kListed];               // thread | number << 16
  float most[kCells][kThreads];         // the greatest logit of each cell
};

__device__ __forceinline__ void offer(Candidates& c, uint64_t key) {
  const uint32_t at = atomicAdd(&c.count, 1u);
  if (at < kCapacity) c.keys[at] = key;
}

// Sets the threshold to the top-th greatest of the groups' greatest keys (0 when fewer groups hold a key). `best` is
// this thread's greatest key. Ends with every thread seeing the threshold. A handful of alternatives is served by
// half as many groups.
__device__ __forceinline__ void set_threshold(Candidates& c, uint64_t best, uint32_t top) {
  const uint32_t lanes = top <= 8 ? 2 * kLanes : kLanes, groups = kThreads / lanes;
  for (uint32_t o = 1; o < lanes; o <<= 1) {
    const uint64_t other = __shfl_xor_sync(0xFFFFFFFFu, best, o);
    best = other > best ? other : best;
  }
  if (threadIdx.x % lanes == 0) c.group[threadIdx.x / lanes] = best;
  if (threadIdx.x == 0) c.threshold = 0;
  __syncthreads();
  const uint64_t own = c.group[threadIdx.x / lanes];
  uint32_t above = 0;  // the lanes of a group share the counting
#pragma unroll 4
  for (uint32_t i = threadIdx.x % lanes; i < groups; i += lanes) above += c.group[i] > own ? 1u : 0u;
  for (uint32_t o = 1; o < lanes; o <<= 1) above += __shfl_xor_sync(0xFFFFFFFFu, above, o);
  if (above == top - 1 && own != 0) c.threshold = own;  // keys differ: one group at most
  __syncthreads();
}

// The lanes whose greatest logits make one group, from which the bar is taken.
__device__ __forceinline__ uint32_t group_lanes(uint32_t top) { return top <= 8 ? 2 * kLanes : kLanes; }

// Publishes the greatest logit of each group.
__device__ __forceinline__ float group_greatest(Candidates& c, float greatest, uint32_t top) {
  const uint32_t lanes = group_lanes(top);
  for (uint32_t o = 1; o < lanes; o <<= 1) greatest = fmaxf(greatest, __shfl_xor_sync(0xFFFFFFFFu, greatest, o));
  if (threadIdx.x % lanes == 0) reinterpret_cast<float*>(c.group)[threadIdx.x / lanes] = greatest;
  return greatest;
}

// Sets the bar to the top-th greatest of the groups' greatest logits, a lower bound on the top-th greatest of them all.
__device__ __forceinline__ void set_bar(Candidates& c, float greatest, uint32_t top) {
  const uint32_t lanes = group_lanes(top), groups = kThreads / lanes;
  const float* group = reinterpret_cast<const float*>(c.group);
  uint32_t above = 0, from = 0;  // groups above this one's, and at or above it
#pragma unroll 4
  for (uint32_t i = threadIdx.x % lanes; i < groups; i += lanes) {
    above += group[i] > greatest ? 1u : 0u;
    from += group[i] >= greatest ? 1u : 0u;
  }
  for (uint32_t o = 1; o < lanes; o <<= 1) {
    above += __shfl_xor_sync(0xFFFFFFFFu, above, o);
    from += __shfl_xor_sync(0xFFFFFFFFu, from, o);
  }
  if (above < top && from >= top) c.bar = greatest;  // (groups that write it write the same)
}

// Drops candidates that cannot be among the `top` greatest: at most `top` groups hold a key at or above the threshold,
// so n keys leave at most top * lanes * ceil(n / kThreads), which is less while n > kThreads. Called by the whole CTA,
// with the list settled and not overflown.
__device__ __noinline__ void thin(Candidates& c, uint32_t top) {
  constexpr uint32_t kPer = kCapacity / kThreads;
  const uint32_t count = c.count;
  uint64_t own[kPer], best = 0;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i) {
    const uint32_t at = i * kThreads + threadIdx.x;
    own[i] = at < count ? c.keys[at] : 0;
    best = own[i] > best ? own[i] : best;
  }
  set_threshold(c, best, top);
  if (threadIdx.x == 0) c.count = 0;
  __syncthreads();
  const uint64_t threshold = c.threshold;
#pragma unroll
  for (uint32_t i = 0; i < kPer; ++i)
    if (own[i] != 0 && own[i] >= threshold) c.keys[atomicAdd(&c.count, 1u)] = own[i];
  __syncthreads();
}

// A part of the row: l = sum 2^(y - m) and t = sum (y - m) 2^(y - m) over its logits in bits, y = x log2 e. One fused
// multiply-add gives y - m, rounded once; m is whatever reference the products were taken against, so its own rounding
// cancels. That rounding grows with the logit, though, and 2^(y - m) with it. So logits at or below kDeep (masks) count
// for nothing: floats above it lie at least 64 above, beside which they weigh e^-64; and a row whose reference is
// beyond kLarge, or that has nothing above kDeep (l = 0), is summed again in plain units (plain_sums).
constexpr float kDeep = -0x1p30f, kLarge = 0x1p24f;
struct Sums {
  float m, l, t;
};
__device__ __forceinline__ Sums no_sums() { return Sums{2.f * kDeep, 0.f, 0.f}; }

// The sums of both at the greater reference: with y - m' = (y - m) + (m - m').
__device__ __forceinline__ Sums merge(const Sums& a, const Sums& b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float da = a.m - r.m, db = b.m - r.m, fa = fast_exp2(da), fb = fast_exp2(db);
  r.l = a.l * fa + b.l * fb;
  r.t = fmaf(da, a.l, a.t) * fa + fmaf(db, b.l, b.t) * fb;
  return r;
}

// The warp's sums: one rescaling to its maximum, then plain additions.
__device__ __forceinline__ Sums warp_merge(Sums s) {
  float m = s.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  const float d = s.m - m, f = fast_exp2(d);
  return Sums{m, warp_sum(s.l * f), warp_sum(fmaf(d, s.l, s.t) * f)};
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_rank(const void* local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
  return remote;
}
__device__ __forceinline__ float ld_rank(const float* local, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(in_rank(local, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t ld_rank(const uint64_t* local, uint32_t rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(in_rank(local, rank)) : "memory");
  return v;
}

// Moves the reference up to the logit `most`.
__device__ __forceinline__ void raise(Sums& s, float most) {
  const float m = most * kLog2e;
  if (m > s.m) {
    const float d = s.m - m, f = fast_exp2(d);
    s.t = fmaf(d, s.l, s.t) * f;
    s.l *= f;
    s.m = m;
  }
}

__device__ __forceinline__ void add_one(Sums& s, float x) {
  if (x <= kDeep) return;
  raise(s, x);
  const float y = fmaf(x, kLog2e, -s.m), e = fast_exp2(y);
  s.l += e;
  s.t = fmaf(y, e, s.t);
}

// The running sums over the logits of N words; returns the greatest of them.
template <typename T, uint32_t N>
__device__ __forceinline__ float add(Sums& s, const uint32_t (&w)[N]) {
  constexpr uint32_t kPairs = N * Logits<T>::kPerWord / 2;
  float most, least;
  Logits<T>::range(w, most, least);
  raise(s, most);  // (a reference below every logit that counts stays)
  if (least > kDeep) {
    const uint64_t base = f2_splat(-s.m), scale = f2_splat(kLog2e);
    uint64_t l = f2_splat(0.f), t = f2_splat(0.f);
#pragma unroll
    for (uint32_t j = 0; j < kPairs; ++j) {
      float a, b;
      Logits<T>::pair(w, j, a, b);
      const uint64_t y = f2_fma(f2_pack(a, b), scale, base);
      f2_unpack(y, a, b);
      const uint64_t e = f2_pack(fast_exp2(a), fast_exp2(b));
      l = f2_add(l, e);
      t = f2_fma(y, e, t);
    }
    float l0, l1, t0, t1;
    f2_unpack(l, l0, l1);
    f2_unpack(t, t0, t1);
    s.l += l0 + l1;
    s.t += t0 + t1;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 2 * kPairs; ++j) {
      float a, b;
      Logits<T>::pair(w, j / 2, a, b);
      const float x = j % 2 ? b : a, y = fmaf(x <= kDeep ? kDeep : x, kLog2e, -s.m);
      const float e = x <= kDeep ? 0.f : fast_exp2(y);
      s.l += e;
      s.t = fmaf(y, e, s.t);
    }
  }
  return most;
}

// A row's sums by one CTA in the plain units of the logits: d = x - greatest, the sums of e^d and d e^d (NaN when the row
// holds a NaN or +infinity; 0 when it holds nothing but -infinity). The greatest ignores NaN, so a row of NaN and -infinity
// alone is told apart by looking for one.
template <typename T>
__device__ __noinline__ Sums plain_sums(const T* row, uint32_t vocab, Sums* scratch) {
  Sums s{-INFINITY, 0.f, 0.f};
  bool nan = false;
  for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
    const float x = Logits<T>::one(row + i);
    nan = nan || x != x;
    s.m = fmaxf(s.m, x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s.m = fmaxf(s.m, __shfl_xor_sync(0xFFFFFFFFu, s.m, o));
  __syncthreads();
  if (lane_id() == 0) scratch[warp_id()].m = s.m;
  nan = __syncthreads_or(nan);
  for (uint32_t w = 0; w < kWarps; ++w) s.m = fmaxf(s.m, scratch[w].m);
  if (s.m == -INFINITY) {
    if (nan) s.l = s.t = __int_as_float(0x7FC00000);
    return s;
  }
  for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
    const float below = Logits<T>::one(row + i) - s.m, d = below < -1000.f ? -1000.f : below, e = fast_exp2(d * kLog2e);
    s.l += e;
    s.t = fmaf(d, e, s.t);
  }
  s.l = warp_sum(s.l);
  s.t = warp_sum(s.t);
  __syncthreads();
  if (lane_id() == 0) scratch[warp_id()] = s;
  __syncthreads();
  s.l = s.t = 0.f;
  for (uint32_t w = 0; w < kWarps; ++w) {
    s.l += scratch[w].l;
    s.t += scratch[w].t;
  }
  return s;
}

// A cluster of `chunks` CTAs per row, each taking a contiguous share of its 16-byte words. TOP: alternatives wanted.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(LogprobParams p) {
  using V = Logits<T>;
  constexpr uint32_t kN = 4 * V::kPerWord;  // logits of a 16-byte word
  extern __shared__ __align__(16) uint8_t raw[];
  Candidates& c = *reinterpret_cast<Candidates*>(raw);
  __shared__ Sums warp_sums[kWarps];
  __shared__ Sums cta_sums;
  __shared__ uint64_t sorted[kMaxTop];
  const uint32_t chunks = p.chunks, chunk = chunks > 1 ? cluster_rank() : 0u, r = blockIdx.x / chunks;
  if (TOP && threadIdx.x == 0) c.count = c.cells = 0;
  if (TOP && threadIdx.x < kMaxTop) sorted[threadIdx.x] = 0;
  pdl_launch_dependents();
  pdl_wait();

  // The row: up to kN - 1 logits before its first 16-byte word, the words, up to kN - 1 logits behind them.
  const T* row = static_cast<const T*>(p.logits) + size_t(r) * p.ld;
  const uint32_t lead = uint32_t((16 - (reinterpret_cast<uintptr_t>(row) & 15u)) & 15u) / sizeof(T);
  const uint32_t head = lead < p.vocab ? lead : p.vocab;
  const uint32_t words = (p.vocab - head) / kN, tail = p.vocab - head - words * kN;
  const uint4* body = reinterpret_cast<const uint4*>(row + head);
  const uint32_t per = (words + chunks - 1) / chunks;
  const uint32_t begin = min(words, chunk * per), end = min(words, begin + per);

  Sums s = no_sums();
  const uint32_t full = (end - begin) / kChunk;  // whole chunks; fewer than kChunk words follow them
  uint4 next[kVectors];
  auto load = [&](uint32_t i) {
    const uint4* at = body + begin + i * kChunk + threadIdx.x;
#pragma unroll
    for (uint32_t v = 0; v < kVectors; ++v)
      if (i < full || begin + i * kChunk + v * kThreads + threadIdx.x < end) next[v] = ld_once(at + v * kThreads);
  };
  load(0);
  const bool reports = chunk == 0 && threadIdx.x == 0;
  const uint32_t id = reports ? uint32_t(p.ids[r]) : 0xFFFFFFFFu;
  // The first CTA takes the logits before the first word and the last one those behind the last, one to a thread.
  const bool edge = (chunk == 0 && threadIdx.x < head) || (chunk == chunks - 1 && threadIdx.x - kN < tail);
  const uint32_t edge_index = threadIdx.x < kN ? threadIdx.x : head + words * kN + threadIdx.x - kN;
  float edge_logit = -INFINITY;
  if (edge) {
    edge_logit = V::one(row + edge_index);
    add_one(s, edge_logit);
  }
  float highest = edge_logit;  // the greatest of this thread's logits
  const uint32_t stride = (end - begin + kChunk * kCells - 1) / (kChunk * kCells);  // chunks of a cell
  uint32_t cell = 0, in_cell = 0;
  float most = -INFINITY;
  auto close = [&]() {  // the cell is complete
    c.most[cell++][threadIdx.x] = most;
    highest = fmaxf(highest, most);
    most = -INFINITY;
    in_cell = 0;
  };
  for (uint32_t i = 0; i < full; ++i) {
    uint32_t w[4 * kVectors];
#pragma unroll
    for (uint32_t v = 0; v < kVectors; ++v) {
      w[4 * v] = next[v].x;
      w[4 * v + 1] = next[v].y;
      w[4 * v + 2] = next[v].z;
      w[4 * v + 3] = next[v].w;
    }
    load(i + 1);
    most = fmaxf(most, add<T>(s, w));
    if (TOP && ++in_cell == stride) close();
  }
  // The words behind the whole chunks, one of each thread at a time, as far as the warp has any.
#pragma unroll
  for (uint32_t v = 0; v < kVectors; ++v) {
    const uint32_t at = begin + full * kChunk + v * kThreads + threadIdx.x;
    if (at - lane_id() >= end) break;
    const bool in = at < end;
    const uint32_t w[4] = {in ? next[v].x : V::kMasked, in ? next[v].y : V::kMasked, in ? next[v].z : V::kMasked,
                           in ? next[v].w : V::kMasked};
    most = fmaxf(most, add<T>(s, w));
  }
  if (TOP && (in_cell > 0 || begin + full * kChunk < end)) close();

  const float given = id < p.vocab ? V::one(row + id) : 0.f;  // the given token's logit, on its way meanwhile
  s = warp_merge(s);
  if (lane_id() == 0) warp_sums[warp_id()] = s;
  float group = 0.f;
  if (TOP) group = group_greatest(c, highest, p.top);
  const bool regular = !__syncthreads_or(s.l != s.l);  // no NaN and no infinity
  // The last warp sums up while the others look for the alternatives.
  auto finish_sums = [&]() {
    if (threadIdx.x >= kThreads - 32) {
      s = warp_merge(lane_id() < kWarps ? warp_sums[lane_id()] : no_sums());
      if (lane_id() == 0) cta_sums = s;
    }
  };
  if (!TOP) finish_sums();
  if (TOP) {
    if (regular) {
      set_bar(c, group, p.top);
      __syncthreads();
      const float bar = c.bar;
      if (highest >= bar) {
        for (uint32_t j = 0; j < cell; ++j)
          if (c.most[j][threadIdx.x] >= bar) {
            const uint32_t at = atomicAdd(&c.cells, 1u);
            if (at < kListed) c.cell[at] = threadIdx.x | j << 16;
          }
      }
      if (edge && edge_logit >= bar) offer(c, order_key(edge_logit, edge_index));
      finish_sums();
      __syncthreads();
      const uint32_t steps = stride * kVectors, items = min(c.cells, kListed) * steps;
      for (uint32_t k = threadIdx.x; k < items; k += kThreads) {
        const uint32_t which = c.cell[k / steps];
        const uint32_t at = begin + ((which >> 16) * steps + k % steps) * kThreads + (which & 0xFFFFu);
        if (at >= end) continue;
        if (*reinterpret_cast<volatile uint32_t*>(&c.count) > kCapacity) break;
        const uint4 word = ld_once(body + at);
        const uint32_t w[4] = {word.x, word.y, word.z, word.w};
#pragma unroll
        for (uint32_t i = 0; i < kN; i += 2) {
          float a, b;
          V::pair(w, i / 2, a, b);
          if (a >= bar) offer(c, order_key(a, head + at * kN + i));
          if (b >= bar) offer(c, order_key(b, head + at * kN + i + 1));
        }
      }
    }
    if (!regular) finish_sums();
    __syncthreads();
    if (!regular || c.count > kCapacity || c.cells > kListed) {
      // Rounds of eight logits a thread: most add nothing once the threshold stands; the others go in one by one, with
      // the list thinned and the threshold raised whenever it fills up.
      __syncthreads();
      if (threadIdx.x == 0) {
        c.count = 0;
        c.threshold = 0;
      }
      __syncthreads();
      const uint32_t from = chunk == 0 ? 0 : head + begin * kN;
      const uint32_t to = chunk == chunks - 1 ? p.vocab : head + end * kN;
      for (uint32_t i0 = from; i0 < to; i0 += 8 * kThreads) {
        uint64_t key[8];
        bool any = false;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          const uint32_t i = i0 + j * kThreads + threadIdx.x;
          key[j] = i < to ? order_key(V::one(row + i), i) : 0;
          any = any || key[j] > c.threshold;
        }
        if (!__syncthreads_or(any)) continue;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          if (key[j] > c.threshold) c.keys[atomicAdd(&c.count, 1u)] = key[j];
          __syncthreads();
          while (c.count > kThin) thin(c, p.top);
          __syncthreads();
        }
      }
    }
  }
  // Its greatest keys in order: a short list, in which each candidate counts those above it. (`sorted` is empty before.)
  auto sort = [&]() {
    if (c.count > kThreads / 4) thin(c, p.top);
    while (c.count > kThreads) thin(c, p.top);
    const uint32_t count = c.count;
    // A short list leaves several lanes to each candidate, which share the counting.
    const uint32_t lanes = count <= kThreads / 8 ? 8 : count <= kThreads / 4 ? 4 : count <= kThreads / 2 ? 2 : 1;
    const uint32_t at = threadIdx.x / lanes;
    const uint64_t own = at < count ? c.keys[at] : 0;
    uint32_t above = 0;
    if (at < count) {
#pragma unroll 4
      for (uint32_t k = threadIdx.x % lanes; k < count; k += lanes) above += c.keys[k] > own ? 1u : 0u;
    }
    for (uint32_t o = 1; o < lanes; o <<= 1) above += __shfl_xor_sync(0xFFFFFFFFu, above, o);
    if (at < count && above < p.top) sorted[above] = own;
    __syncthreads();
  };
  if (TOP) sort();
  else __syncthreads();

  if (chunks > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (chunk == 0) {
      s = Sums{ld_rank(&cta_sums.m, 0), ld_rank(&cta_sums.l, 0), ld_rank(&cta_sums.t, 0)};
      for (uint32_t k = 1; k < chunks; ++k)
        s = merge(s, Sums{ld_rank(&cta_sums.m, k), ld_rank(&cta_sums.l, k), ld_rank(&cta_sums.t, k)});
      if (TOP) {
        if (threadIdx.x == 0) c.count = 0;
        __syncthreads();
        for (uint32_t k = threadIdx.x; k < chunks * kMaxTop; k += kThreads) {
          const uint64_t key = ld_rank(&sorted[k % kMaxTop], k / kMaxTop);
          if (key != 0) c.keys[atomicAdd(&c.count, 1u)] = key;
        }
        __syncthreads();
      }
    }
    // No CTA leaves while the first may still read its shared memory.
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (chunk != 0) return;
    if (TOP) sort();
  } else {
    s = cta_sums;
  }

  const bool plain = s.l == 0.f || fabsf(s.m) > kLarge;
  if (plain) s = plain_sums<T>(row, p.vocab, warp_sums);  // (uniform: every thread has the row's sums)
  const bool empty = plain && s.l == 0.f;
  const float log_l = logf(s.l), unit = plain ? 1.f : kLn2;
  auto log_probability = [&](float x) {
    if (empty) return -INFINITY;
    if (plain) return x - s.m - log_l;
    // (a logit of the type's lowest value would overflow in bits)
    return x < -1e30f ? x - fmaf(s.m, kLn2, log_l) : fmaf(fmaf(x, kLog2e, -s.m), kLn2, -log_l);
  };
  uint64_t to = r;
  if (p.slot_of != nullptr) {
    const int64_t slot = int64_t(p.slot_of[r]) + p.slot_offset;
    if (slot < 0 || slot >= int64_t(p.slots)) return;
    to = uint64_t(slot) * p.rows + r;
  }
  if (reports) {
    p.logprob[to] = id >= p.vocab ? 0.f : log_probability(given);
    p.entropy[to] = empty ? 0.f : log_l - unit * (s.t / s.l);
  }
  if (TOP && threadIdx.x < p.top) {
    const uint64_t key = sorted[threadIdx.x];
    p.top_ids[to * p.top + threadIdx.x] = int32_t(0xFFFFFFFFu - uint32_t(key));
    p.top_logprob[to * p.top + threadIdx.x] = log_probability(key_logit(key));
  }
}

template <typename T, bool TOP>
tempo_status launch_logprobs(const LogprobParams& base, cudaStream_t stream) {
  LogprobParams p = base;
  const uint32_t rows = p.rows;
  constexpr uint32_t kBytes = TOP ? sizeof(Candidates) : 0;
  auto kernel = token_logprobs_kernel<T, TOP>;
  tempo_status status = set_smem(reinterpret_cast<const void*>(kernel), kBytes);
  if (status != TEMPO_OK) return status;
  // At most a row for two SMs: a cluster for each, every CTA with at least 1024 logits.
  p.chunks = 1;
  while (p.chunks < kMaxChunks && uint64_t(rows) * p.chunks * 2 <= uint64_t(sm_count()) &&
         p.vocab >= 2 * p.chunks * 1024)
    p.chunks *= 2;
  if (uint64_t(rows) * p.chunks > 0x7FFFFFFFull)
    return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: %u rows are too many for one call", rows);
  return launch(kernel, dim3(rows * p.chunks), dim3(kThreads), kBytes, stream, p.chunks, "token_logprobs_kernel", p);
}

}  // namespace
}  // namespace tempo

using namespace tempo;

extern "C" tempo_status tempo_token_logprobs(const void* logits, uint64_t ld, uint32_t bf16, const int32_t* ids,
                                             uint32_t rows, uint32_t vocab, uint32_t top, float* logprob,
                                             float* entropy, float* top_logprob, int32_t* top_ids,
                                             const int32_t* slot_of, int32_t slot_offset, uint32_t slots,
                                             void* stream) {
  if (rows == 0 || vocab == 0 || vocab > 0x7FFFFFFFu || rows > 0x7FFFFFFFu || ld < vocab)
    return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: rows %u vocab %u, row stride %llu (at least the vocabulary)", rows,
                vocab, static_cast<unsigned long long>(ld));
  if (top > kMaxTop || top > vocab)
    return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: %u alternatives of %u tokens (at most %u)", top, vocab, kMaxTop);
  if (bf16 > 1) return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: the logits are FP32 (0) or BF16 (1), got %u", bf16);
  if (logits == nullptr || (reinterpret_cast<uintptr_t>(logits) & (bf16 ? 1u : 3u)) || ids == nullptr ||
      logprob == nullptr || entropy == nullptr || (top > 0 && (top_logprob == nullptr || top_ids == nullptr)))
    return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: aligned logits, ids and every output are needed");
  if (slot_of != nullptr && slots == 0) return fail(TEMPO_ERR_VALUE, "tempo_token_logprobs: no slots to write to");
  const LogprobParams p{logits, ld, ids, rows, vocab, top, 1, logprob, entropy, top_logprob, top_ids, slot_of, slot_offset,
                        slots};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (bf16) return top > 0 ? launch_logprobs<uint16_t, true>(p, st) : launch_logprobs<uint16_t, false>(p, st);
  return top > 0 ? launch_logprobs<float, true>(p, st) : launch_logprobs<float, false>(p, st);
}
