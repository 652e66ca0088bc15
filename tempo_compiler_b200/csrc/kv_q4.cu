// The 4-bit key/value cache: storing rows of a QKV projection into it, reading rows back, and decode attention over it.
// Each row of 64 dimensions keeps its least value (exact in BF16) and a BF16 scale, so a position costs 72 bytes per
// head and 64 dimensions for key and value together, against 256 in BF16.
#include <algorithm>

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "decode_math.cuh"
#include "host.hpp"
#include "kv_q4.cuh"

namespace tempo {

TEMPO_WATCHDOG_READER(watchdog_kv_q4)

namespace {

constexpr uint32_t kStoreThreads = 128;
constexpr uint32_t kUnitLanes = 4;  // lanes that share a position's 64 dimensions of one key / value head, 16 each
constexpr uint32_t kStoreRows = kStoreThreads / kUnitLanes;

// Rows of keys and values (bf16, `ld` elements apart) and their places in a cache.
struct Q4Rows {
  uint16_t* rows;
  uint8_t* cache;
  const int32_t* seq_of;
  const int32_t* pos_of;
  uint32_t ld, count, seqs, kv_heads, tiles;
};

// A unit: the 64 dimensions of a row's key and of its value that one block holds (group `of` of the row's key groups: the
// key's columns 64 `of` on, the value's as far behind all keys) and where they are kept. A warp takes the same columns of
// eight rows: of a prompt, 256 bytes of codes side by side. (Key and value as two units made the index arithmetic a third of
// the instructions: 116 us for 65536 rows of 12 heads stored and read back instead of 102; with units counted in one grid
// dimension and divided out again 98 instead of 95.)
template <int G>
struct Q4Unit {
  uint32_t row, of, seq, pos;
  __device__ __forceinline__ explicit Q4Unit(const Q4Rows& p) {
    of = blockIdx.x;
    row = blockIdx.y * kStoreRows + threadIdx.x / kUnitLanes;
    seq = pos = 0;
    if (row < p.count) {
      seq = uint32_t(p.seq_of[row]);
      pos = uint32_t(p.pos_of[row]);
    }
  }
  // The unit's block, or null when the place is outside the cache.
  __device__ __forceinline__ uint8_t* place(const Q4Rows& p) const {
    if (seq >= p.seqs || pos >= p.tiles * kQ4Tile) return nullptr;
    return p.cache + q4_block(seq, of / G, pos, of % G, p.kv_heads, p.tiles, G);
  }
  // Lane li's 16 dimensions of the key (0) or the value (1) in a row.
  __device__ __forceinline__ uint4* columns(const Q4Rows& p, uint32_t value, uint32_t li) const {
    return reinterpret_cast<uint4*>(p.rows + size_t(row) * p.ld + (value * gridDim.x + of) * kQ4Group) + 2 * li;
  }
  __device__ __forceinline__ uint2* codes(uint8_t* block, uint32_t value, uint32_t li) const {
    return reinterpret_cast<uint2*>(block + value * kQ4Codes + pos % kQ4Tile * 32) + li;
  }
  __device__ __forceinline__ uint2* meta(uint8_t* block) const {
    return reinterpret_cast<uint2*>(block + 2 * kQ4Codes) + pos % kQ4Tile;
  }
};

__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t min_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Eight codes as a word, the first in its lowest bits, from the floats 1.5 2^23 + code: these hold the code in their lowest
// four bits and nothing in the eighteen above.
__device__ __forceinline__ uint32_t pack_codes(const uint32_t* c) {
  const uint32_t b01 = __byte_perm(c[1] * 16 + c[0], c[3] * 16 + c[2], 0x0040);
  const uint32_t b23 = __byte_perm(c[5] * 16 + c[4], c[7] * 16 + c[6], 0x0040);
  return __byte_perm(b01, b23, 0x5410);
}

// Storing is bound by the bytes it moves as long as the arithmetic stays near ten instructions a value. The least and
// greatest value come from packed BF16 comparisons (a NaN stays); scale = bf16((greatest - least) / 15); and the
// code is the quotient (x - least) / scale, correctly rounded to FP32, rounded to the nearest integer, ties to even. With
// r = 1 / scale correctly rounded, q = d r and q + (d - q scale) r is the correctly rounded quotient (Markstein's
// theorem) while nothing underflows; scales outside [2^-90, 2^100] take the division itself. Adding 1.5 2^23 rounds.
// A row of values that are all equal has scale 0 and codes 0; one with a NaN, an infinity or a range that
// passes FP32 has a scale that is not finite, and reads back as NaN. (A first form, eight lanes to a row with a 64-bit
// index division, FP32 divisions and conversions, took 304 us for storing and reading 65536 rows of 12 heads.)
__device__ __forceinline__ uint2 quantise(const uint4& a, const uint4& b, uint32_t mask, uint32_t& meta) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t most = w[0], least = w[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    most = max_nan_bf16x2(most, w[i]);
    least = min_nan_bf16x2(least, w[i]);
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    most = max_nan_bf16x2(most, __shfl_xor_sync(mask, most, o));
    least = min_nan_bf16x2(least, __shfl_xor_sync(mask, least, o));
  }
  // both halves of each word
  most = max_nan_bf16x2(most, __byte_perm(most, 0, 0x1032));
  least = min_nan_bf16x2(least, __byte_perm(least, 0, 0x1032));
  const float high = bf16_lo(most), low = bf16_lo(least);
  const bool finite = fabsf(high) < INFINITY && fabsf(low) < INFINITY;  // false for a NaN too
  const float scale = finite ? round_bf16(__fdiv_rn(high - low, 15.f)) : __int_as_float(0x7FC00000);
  uint32_t c[16];
  if (scale >= 0x1p-90f && scale <= 0x1p100f) {
    const float r = __frcp_rn(scale);
    const uint64_t r2 = f2_splat(r), s2 = f2_splat(-scale), low2 = f2_splat(-low), round2 = f2_splat(12582912.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t d = f2_add(f2_pack(bf16_lo(w[i]), bf16_hi(w[i])), low2);
      const uint64_t q = f2_mul(d, r2);
      const uint64_t exact = f2_fma(f2_fma(q, s2, d), r2, q);
      // in 0 .. 15: the scale's rounding moves a quotient by at most 15 / 256
      float c0, c1;
      f2_unpack(f2_add(exact, round2), c0, c1);
      c[2 * i] = __float_as_uint(c0);
      c[2 * i + 1] = __float_as_uint(c1);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = i % 2 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
      const float code = scale > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x - low, scale)), 0.f), 15.f) : 0.f;
      c[i] = __float_as_uint(code + 12582912.f);
    }
  }
  meta = pack_bf16x2(scale, finite ? low : 0.f);
  return make_uint2(pack_codes(c), pack_codes(c + 8));
}

// 16 dimensions of a row, 32 bytes: one access where rows begin on 32 bytes (WIDE: reading back 65536 rows 46.5 us), else two
// of 16, each of half a sector (49.8).
template <bool WIDE>
__device__ __forceinline__ void load_columns(const uint4* p, uint4& a, uint4& b) {
  if constexpr (WIDE) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
                 : "l"(p));
  } else {
    a = p[0];
    b = p[1];
  }
}
template <bool WIDE>
__device__ __forceinline__ void store_columns(uint4* p, const uint4& a, const uint4& b) {
  if constexpr (WIDE) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
                 "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
  } else {
    p[0] = a;
    p[1] = b;
  }
}

template <int G, bool WIDE>
__global__ void __launch_bounds__(kStoreThreads) kv_store_q4_kernel(Q4Rows p) {
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t li = threadIdx.x % kUnitLanes, mask = 0xFu << (threadIdx.x & 28u);
  const Q4Unit<G> unit(p);
  if (unit.row >= p.count) return;  // whole units leave together
  // The row is on its way before its place is known; a place outside the cache only keeps it from being stored.
  uint4 k0, k1, v0, v1;
  load_columns<WIDE>(unit.columns(p, 0, li), k0, k1);
  load_columns<WIDE>(unit.columns(p, 1, li), v0, v1);
  uint8_t* block = unit.place(p);
  uint2 meta;
  const uint2 k = quantise(k0, k1, mask, meta.x), v = quantise(v0, v1, mask, meta.y);
  if (block == nullptr) return;
  *unit.codes(block, 0, li) = k;
  *unit.codes(block, 1, li) = v;
  if (li == 0) *unit.meta(block) = meta;
}

// The rows' keys and values back as BF16: code x scale + low in FP32, rounded once.
template <int G, bool WIDE>
__global__ void __launch_bounds__(kStoreThreads) kv_load_q4_kernel(Q4Rows p) {
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t li = threadIdx.x % kUnitLanes;
  const Q4Unit<G> unit(p);
  if (unit.row >= p.count) return;
  uint8_t* block = unit.place(p);
  uint2 codes[2] = {make_uint2(0, 0), make_uint2(0, 0)}, meta = make_uint2(0, 0);  // a place outside the cache: zeros
  if (block != nullptr) {
    codes[0] = *unit.codes(block, 0, li);
    codes[1] = *unit.codes(block, 1, li);
    meta = *unit.meta(block);
  }
#pragma unroll
  for (uint32_t value = 0; value < 2; ++value) {
    const uint32_t words = value ? meta.y : meta.x;
    const float s = bf16_lo(words), l = bf16_hi(words);
    uint32_t out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t word = (i < 4 ? codes[value].x : codes[value].y) >> (8 * (i % 4));
      // a code under the exponent of 2^23 is the float 2^23 + code
      const float c0 = __uint_as_float((word & 15u) | 0x4B000000u) - 8388608.f;
      const float c1 = __uint_as_float(((word >> 4) & 15u) | 0x4B000000u) - 8388608.f;
      out[i] = pack_bf16x2(fmaf(c0, s, l), fmaf(c1, s, l));
    }
    store_columns<WIDE>(unit.columns(p, value, li), make_uint4(out[0], out[1], out[2], out[3]),
                        make_uint4(out[4], out[5], out[6], out[7]));
  }
}

// Rows that all begin on 32 bytes.
bool wide_rows(const Q4Rows& p) { return reinterpret_cast<uintptr_t>(p.rows) % 32 == 0 && p.ld % 16 == 0; }

// Launches `kernel` over `rows` rows, in as many calls as the grid's 16-bit dimension needs.
tempo_status launch_rows(void (*kernel)(Q4Rows), Q4Rows p, uint32_t rows, uint32_t groups, cudaStream_t stream,
                         const char* name) {
  for (uint32_t done = 0; done < rows;) {
    p.count = std::min(rows - done, 65535 * kStoreRows);
    const tempo_status status = launch(kernel, dim3(p.kv_heads * groups, (p.count - 1) / kStoreRows + 1),
                                       dim3(kStoreThreads), 0, stream, 1, name, p);
    if (status != TEMPO_OK) return status;
    p.rows += size_t(p.count) * p.ld;
    p.seq_of += p.count;
    p.pos_of += p.count;
    done += p.count;
  }
  return TEMPO_OK;
}

// ---------------------------------------------------------------------------------------------------------------
// Decode attention
//
// At 72 bytes a position the cache streams past at more than 40 codes per clock and SM, which CUDA cores cannot
// dequantise, multiply and add in FP32 (a first kernel that did so took 4 to 150 times the read time), so both products
// run on mma.sync with the codes as the A operand: masked where they stand in a 16-bit word, pairs of codes are the FP16
// subnormals code 2^-20, and scale and low are applied to the products: with D = sum_d q_d code_d and Q = sum_d q_d,
//   q . k = scale D + low Q,
//   sum_j p_j v_j = sum_j w_j code_j + sum_j p_j low_j,   w_j = p_j scale_j.
// (As the integers 64 + code, with 64 sum_j w_j taken off again, a warp's sums over 2^18 positions were 2 % of the values' range
// off: the tensor core's additions round towards zero, and 64 sum_j w_j did not round alike.)
// What bounds the kernel is the logic pipe: a code pair costs one logic operation to mask and one to move, of which those
// to the left are multiplications by 16 and run beside them (shifts for all of them, the keys as BF16 integers 128 +
// code, took 91 us for 512 sequences of 12 heads and 1152 positions instead of 89.6; moves to the right as the high half
// of a product, in place of the byte swaps, 104 instead of 85). The values come through the transposing matrix load,
// which puts the same dimensions of two positions side by side (85 us; byte permutations for it took 89). It now takes 77.3 us,
// 0.96 of the measured copy rate; two sequences of 32 query heads over 8 of 128 and 40001 to 65536 positions 35.7.
// The eight columns of the B operand (m16n8k16) are query heads of one key / value head times tiles:
// grouped heads read the cache once, and with few heads one softmax serves several tiles (the first tensor-core form, one tile
// and eight columns of queries whether they existed or not, issued 309 instructions a tile and was bound by the ALU pipe).
// Every column holds its head's query; the scores of tile j are kept in the lanes whose columns are tile j's, and the
// weights of the other columns are zeroed before tile j's values are multiplied.
// Each 64 dimensions of a query row are scaled by a power of two to at most 2, where FP16 holds their BF16 values but for what
// lies 2^-14 below the greatest of them, and there to 2^-25 (as FP32 sums with keys that share a scale would); w is rounded to
// FP16 (2^-11 of each weight, an eighth of the output's own BF16 rounding, and 2^-33 of the greatest), in a running unit that
// bounds w and p low alike; everything else, the sums included, is FP32.
//
// A CTA of two, four or eight warps takes a run of tiles of one (sequence, key / value head, up to eight query heads); each
// warp streams its own pieces (one bulk copy each, kRing in flight) and keeps an online softmax whose reference and units move
// only when a weight passes them some hundred times. Warps merge through shared memory; with `chunks` > 1 the CTAs of a
// cluster split the positions and merge through distributed shared memory, or, when a pair needs more of them, through a
// workspace and a second kernel.
// ---------------------------------------------------------------------------------------------------------------

constexpr uint32_t kQ4MaxChunks = 8;     // CTAs of a cluster
constexpr uint32_t kQ4MaxSplits = 160;   // CTAs that share a pair through the workspace
constexpr uint32_t kQ4Queries = 8;
constexpr uint32_t kQ4Piece = 4 * kQ4Block;  // bytes of one bulk copy: four tiles of a 64-wide head, two of a 128-wide
constexpr uint32_t kRing = 2;
constexpr float kCodeOne = 0x1p20f;  // what makes a code of the A operands' whole
constexpr float kNoScore = -3.4028235e38f;  // the reference before any position: no finite score is below it,
constexpr int kNoUnit = -100;               // and no unit
// The reference is set kLift below the greatest score, so the smallest p = 2^(score - reference), 2^-126, is 2^-150 of the
// greatest, as small as FP32 goes. (Beside large scores their difference rounds to anything from 0 to 32, which is as good.)
constexpr float kLift = 24.f;
// A unit holds the greatest weight it is set for as 2^kTop, so that w = 2^-24, the least that FP16 holds, is 2^-32 of it: what
// that rounds away is half of it a position at most, 2^-13 of the values' range over a million. (At kTop 0 such a tail of weights
// near 2^-25 was lost from the values and not from the sum.)
constexpr float kTop = 8.f;
constexpr float kSlack = 0x1p15f;           // what w may reach before the unit moves (FP16 holds 65504),
constexpr float kSlackP = 0x1p37f;          // and p before the reference does

template <int G, int WARPS>
struct Q4Smem {
  static constexpr uint32_t kWarpRing = kRing * kQ4Piece;
  // A partial result of eight queries: 64 G values each (dimension 64 i + 4 g + n at 64 i + 8 n + g, eight words more to
  // the next query: the lanes of a fragment store into different banks), then the references, the units' exponents
  // (eight of each group) and the sums.
  static constexpr uint32_t kStride = 64 * G + 8;
  static constexpr uint32_t kReferences = kQ4Queries * kStride, kUnits = kReferences + kQ4Queries;
  static constexpr uint32_t kSums = kUnits + G * kQ4Queries;
  static constexpr uint32_t kPart = (kSums + kQ4Queries) * 4;
  static constexpr uint32_t kBarrierOffset = WARPS * kWarpRing;
  static constexpr uint32_t kMergeOffset = kBarrierOffset + WARPS * kRing * 8;
  static constexpr uint32_t kBytes = kMergeOffset + kPart;  // the CTA's own partial result last, for its cluster
  static_assert(kPart <= kWarpRing && kPart % 16 == 0, "a warp's partial result fits its ring");
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// D = A x B: the accumulator starts at zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// D += A x B.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 matrix of 16-bit words held two per lane (row lane / 4, columns 2 (lane % 4) and + 1).
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Four 8 x 8 matrices of 16-bit words, transposed: lane l gives the address of row l % 8 of matrix l / 8.
__device__ __forceinline__ void load_transposed(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d, uint32_t row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
               : "r"(row));
}

__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A constant that the compiler does not know, and keeps in a register.
__device__ __forceinline__ uint32_t in_register(uint32_t c) {
  asm volatile("" : "+r"(c));
  return c;
}

struct Q4Constants {
  uint32_t mask, sixteen;
};

// Two codes as the FP16 subnormals code 2^-20: code 0 or 1 of each half of w (bits 0 .. 3 or 4 .. 7). The multiplier is not
// known to be 16 when the kernel is compiled, so the product stays one, beside the logic pipe.
__device__ __forceinline__ uint32_t pair0(const Q4Constants& k, uint32_t w) { return w * k.sixteen & k.mask; }
__device__ __forceinline__ uint32_t pair1(const Q4Constants& k, uint32_t w) { return w & k.mask; }
// The bytes of each half swapped: codes 2 and 3 where 0 and 1 were.
__device__ __forceinline__ uint32_t swap_bytes(uint32_t w) { return __byte_perm(w, 0, 0x2301); }

// One warp's running state. The MMA fragments put columns 2 t and 2 t + 1 (t = lane % 4) on a lane; with g = lane / 4,
// acc[i][n] holds dimensions 64 i + 4 g + n ([0], [1]) and 32 more ([2], [3]) of the two columns.
template <int G>
struct Q4State {
  float acc[G][4][4];
  float m[2];       // the reference, a score
  float inv[G][2];  // 1 / the unit (a power of two) in which a group's acc and low are counted
  float l[2];       // this lane's sum of p
  float low[G][2];  // this lane's sums of p low
};

__device__ __forceinline__ int unit_exponent(float inv) { return 127 - int(__float_as_uint(inv) >> 23); }
__device__ __forceinline__ float inverse_unit(int exponent) { return __uint_as_float(uint32_t(127 - exponent) << 23); }

// A value row's size: its scale, or a sixteenth of its low where that is more.
__device__ __forceinline__ float q4_size(uint32_t meta) {
  return fmax3(0x1p-100f, bf16_lo(meta), 0.0625f * fabsf(bf16_hi(meta)));
}

__device__ __forceinline__ float q4_weight(float score, float reference) { return fast_exp2(score - reference); }

// Moves a unit to hold weights of 2^x as 2^kTop, and what it held, whose reference rises by -down: returns the factor
// that brings that to the new unit, at most 1.
__device__ __forceinline__ float q4_move(float& inv, float down, float x) {
  const int was = unit_exponent(inv);
  const int now = int(fminf(fmaxf(fmaxf(ceilf(x) - kTop, ceilf(down) + float(was)), float(kNoUnit)), 126.f));
  inv = inverse_unit(now);
  return fast_exp2(down + float(was - now));
}

// Columns of a tile: the RP query heads, or two (the odd one empty) for a single head, which leaves half of each lane's
// softmax out.
__host__ __device__ constexpr uint32_t q4_columns(int rp) { return rp == 1 ? 2u : uint32_t(rp); }
// Tiles of one softmax: 8 columns' worth, at most a piece.
__host__ __device__ constexpr uint32_t q4_tiles_at_once(int g, int rp) {
  return 8 / q4_columns(rp) < 4u / g ? 8 / q4_columns(rp) : 4u / g;
}

// Folds TP tiles in shared memory into the state. FULL: every position of them exists;
// else `left` do.
template <int G, int RP, bool FULL>
__device__ __forceinline__ void q4_tiles(Q4State<G>& st, const uint32_t (&qf)[G][8], const float (&qs)[G][2],
                                         const float (&unit)[G][2],
                                         const uint8_t* tiles, uint32_t left, uint32_t g, uint32_t t,
                                         const Q4Constants& kc) {
  constexpr uint32_t kTileBytes = G * kQ4Block, CP = q4_columns(RP), TP = q4_tiles_at_once(G, RP);
  constexpr bool kTwo = RP > 1;  // a single query takes the even columns only
  // Row r of the score MMA is position pi(r) (r < 8) or 8 + pi(r - 8) of a tile, pi = 0 2 1 3 6 4 7 5: the key words of
  // eight lane groups then fall into different banks.
  const uint32_t pg = g & 1u ? (g >> 1) + 2 : (g < 4 ? g >> 1 : (g >> 1) + 4);
  // Lane l's row of the transposing value load: position pi(l % 8), or 8 + that, and 32 dimensions.
  const uint32_t l8 = lane_id() & 7u, pl = l8 & 1u ? (l8 >> 1) + 2 : (l8 < 4 ? l8 >> 1 : (l8 >> 1) + 4);
  const uint32_t value_rows = smem_u32(tiles) + kQ4Codes + (pl + (lane_id() >> 4) * 8) * 32 + (lane_id() >> 3 & 1u) * 16;
  const uint32_t mine = 2 * t / CP;                   // the tile of this lane's two columns (none when >= TP)
  float d[G][4];
#pragma unroll
  for (int i = 0; i < G; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.f;
#pragma unroll
  for (uint32_t j = 0; j < TP; ++j) {
    if (!FULL && j * kQ4Tile >= left) break;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const uint8_t* block = tiles + j * kTileBytes + i * kQ4Block;
      const uint2 k0 = *reinterpret_cast<const uint2*>(block + pg * 32 + t * 8);
      const uint2 k1 = *reinterpret_cast<const uint2*>(block + (pg + 8) * 32 + t * 8);
      float e[4];
      const uint32_t x0 = swap_bytes(k0.x), x1 = swap_bytes(k1.x), y0 = swap_bytes(k0.y), y1 = swap_bytes(k1.y);
      mma_f16_first(e, pair0(kc, k0.x), pair0(kc, k1.x), pair1(kc, k0.x), pair1(kc, k1.x), qf[i][0], qf[i][1]);
      mma_f16(e, pair0(kc, x0), pair0(kc, x1), pair1(kc, x0), pair1(kc, x1), qf[i][2], qf[i][3]);
      mma_f16(e, pair0(kc, k0.y), pair0(kc, k1.y), pair1(kc, k0.y), pair1(kc, k1.y), qf[i][4], qf[i][5]);
      mma_f16(e, pair0(kc, y0), pair0(kc, y1), pair1(kc, y0), pair1(kc, y1), qf[i][6], qf[i][7]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (kTwo || c % 2 == 0) d[i][c] = TP == 1 || mine == j ? e[c] : d[i][c];
    }
  }
  const bool in0 = (TP == 4 || mine < TP) && (FULL || mine * kQ4Tile + pg < left);
  const bool in1 = (TP == 4 || mine < TP) && (FULL || mine * kQ4Tile + pg + 8 < left);
  const uint8_t* own = tiles + (TP == 4 || mine < TP ? mine : 0u) * kTileBytes + 2 * kQ4Codes;
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;  // scores (log2): rows g and g + 8, columns 2 t and 2 t + 1
  uint32_t vm0[G], vm1[G];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    uint2 meta0 = *reinterpret_cast<const uint2*>(own + i * kQ4Block + pg * 8);
    uint2 meta1 = *reinterpret_cast<const uint2*>(own + i * kQ4Block + (pg + 8) * 8);
    if (!in0) meta0 = make_uint2(0, 0);  // what lies behind the last position may be anything
    if (!in1) meta1 = make_uint2(0, 0);
    const float ks0 = bf16_lo(meta0.x) * kCodeOne, ks1 = bf16_lo(meta1.x) * kCodeOne;
    const float kl0 = bf16_hi(meta0.x), kl1 = bf16_hi(meta1.x);
    s0 = __fmaf_rn(fmaf(ks0, d[i][0], kl0 * qs[i][0]), unit[i][0], s0);
    if (kTwo) s1 = __fmaf_rn(fmaf(ks0, d[i][1], kl0 * qs[i][1]), unit[i][1], s1);
    s2 = __fmaf_rn(fmaf(ks1, d[i][2], kl1 * qs[i][0]), unit[i][0], s2);
    if (kTwo) s3 = __fmaf_rn(fmaf(ks1, d[i][3], kl1 * qs[i][1]), unit[i][1], s3);
    vm0[i] = meta0.y;
    vm1[i] = meta1.y;
  }
  if (!in0) s0 = s1 = -INFINITY;
  if (!in1) s2 = s3 = -INFINITY;
  // The reference follows the scores alone: the sum l of p = 2^(score - reference) keeps every position's share, whatever the
  // values. A group's weights w = p scale and p low are counted in a unit of their own, a power of two that follows p size,
  // size the value row's scale or a sixteenth of its low, so they stay small whatever the values' size and the halves of a
  // head of 128 keep their bits beside one another. Reference and units move when w passes kSlack or p kSlackP (which NaN and
  // infinity do too).
  float p0 = q4_weight(s0, st.m[0]), p2 = q4_weight(s2, st.m[0]);
  float p1 = kTwo ? q4_weight(s1, st.m[1]) : 0.f, p3 = kTwo ? q4_weight(s3, st.m[1]) : 0.f;
  float u0[G], u1[G], u2[G], u3[G], l0 = p0 + p2, l1 = p1 + p3;  // u: p in the groups' units
  auto scale = [&]() {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      u0[i] = p0 * st.inv[i][0];
      u2[i] = p2 * st.inv[i][0];
      u1[i] = kTwo ? p1 * st.inv[i][1] : 0.f;
      u3[i] = kTwo ? p3 * st.inv[i][1] : 0.f;
    }
  };
  scale();
  float far0 = l0 * (kSlack / kSlackP), far1 = l1 * (kSlack / kSlackP);
#pragma unroll
  for (int i = 0; i < G; ++i) {
    far0 = fmaf(u0[i], q4_size(vm0[i]), fmaf(u2[i], q4_size(vm1[i]), far0));
    if (kTwo) far1 = fmaf(u1[i], q4_size(vm0[i]), fmaf(u3[i], q4_size(vm1[i]), far1));
  }
  if (__any_sync(0xFFFFFFFFu, !(far0 <= kSlack) || (kTwo && !(far1 <= kSlack)))) {
    float m0 = fmaxf(s0, s2) - kLift, m1 = kTwo ? fmaxf(s1, s3) - kLift : 0.f;
#pragma unroll
    for (int o = 4; o <= 16; o <<= 1) {
      m0 = fmaxf(m0, __shfl_xor_sync(0xFFFFFFFFu, m0, o));
      if (kTwo) m1 = fmaxf(m1, __shfl_xor_sync(0xFFFFFFFFu, m1, o));
    }
    m0 = fmaxf(m0, st.m[0]);
    if (kTwo) m1 = fmaxf(m1, st.m[1]);
    const float down0 = st.m[0] - m0, down1 = kTwo ? st.m[1] - m1 : 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const float g0 = fast_log2(fminf(q4_size(vm0[i]), 0x1p100f)), g1 = fast_log2(fminf(q4_size(vm1[i]), 0x1p100f));
      float x0 = fmaxf(s0 - m0 + g0, s2 - m0 + g1), x1 = kTwo ? fmaxf(s1 - m1 + g0, s3 - m1 + g1) : 0.f;
#pragma unroll
      for (int o = 4; o <= 16; o <<= 1) {
        x0 = fmaxf(x0, __shfl_xor_sync(0xFFFFFFFFu, x0, o));
        if (kTwo) x1 = fmaxf(x1, __shfl_xor_sync(0xFFFFFFFFu, x1, o));
      }
      const float c0 = q4_move(st.inv[i][0], down0, x0), c1 = kTwo ? q4_move(st.inv[i][1], down1, x1) : 0.f;
      st.low[i][0] *= c0;
      if (kTwo) st.low[i][1] *= c1;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        st.acc[i][n][0] *= c0;
        st.acc[i][n][2] *= c0;
        if (kTwo) {
          st.acc[i][n][1] *= c1;
          st.acc[i][n][3] *= c1;
        }
      }
    }
    st.m[0] = m0;
    st.l[0] *= fast_exp2(down0);
    p0 = q4_weight(s0, m0);
    p2 = q4_weight(s2, m0);
    if (kTwo) {
      st.m[1] = m1;
      st.l[1] *= fast_exp2(down1);
      p1 = q4_weight(s1, m1);
      p3 = q4_weight(s3, m1);
    }
    scale();
    l0 = p0 + p2;
    l1 = p1 + p3;
  }
  st.l[0] += l0;
  if (kTwo) st.l[1] += l1;
  uint32_t b0[G], b1[G];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const float vs0 = bf16_lo(vm0[i]), vs1 = bf16_lo(vm1[i]), vl0 = bf16_hi(vm0[i]), vl1 = bf16_hi(vm1[i]);
    const __half2 h0 = __floats2half2_rn(u0[i] * vs0, kTwo ? u1[i] * vs0 : 0.f);
    const __half2 h1 = __floats2half2_rn(u2[i] * vs1, kTwo ? u3[i] * vs1 : 0.f);
    st.low[i][0] = fmaf(u0[i], vl0, fmaf(u2[i], vl1, st.low[i][0]));
    if (kTwo) st.low[i][1] = fmaf(u1[i], vl0, fmaf(u3[i], vl1, st.low[i][1]));
    b0[i] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h0));
    b1[i] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h1));
  }
#pragma unroll
  for (uint32_t j = 0; j < TP; ++j) {
    if (!FULL && j * kQ4Tile >= left) break;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const uint32_t w0 = TP == 1 || g / CP == j ? b0[i] : 0u, w1 = TP == 1 || g / CP == j ? b1[i] : 0u;
      // The same dimensions of two positions side by side: 4 g .. 4 g + 3 in the first word of each pair, 32 more in the
      // second; codes 0 and 1, and 2 and 3 of each half with its bytes swapped.
      uint32_t e0, o0, e1, o1;
      load_transposed(e0, o0, e1, o1, value_rows + j * kTileBytes + i * kQ4Block);
      const uint32_t f0 = swap_bytes(e0), r0 = swap_bytes(o0), f1 = swap_bytes(e1), r1 = swap_bytes(o1);
      mma_f16(st.acc[i][0], pair0(kc, e0), pair0(kc, o0), pair0(kc, e1), pair0(kc, o1), w0, w1);
      mma_f16(st.acc[i][1], pair1(kc, e0), pair1(kc, o0), pair1(kc, e1), pair1(kc, o1), w0, w1);
      mma_f16(st.acc[i][2], pair0(kc, f0), pair0(kc, r0), pair0(kc, f1), pair0(kc, r1), w0, w1);
      mma_f16(st.acc[i][3], pair1(kc, f0), pair1(kc, r0), pair1(kc, f1), pair1(kc, r1), w0, w1);
    }
  }
}

__device__ __forceinline__ float ld_cluster(const float* local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}

// The dimension of word `at` of a query's values in a partial result.
__device__ __forceinline__ uint32_t q4_dimension(uint32_t at) { return (at & ~31u) | (at & 7u) << 2 | (at >> 3 & 3u); }

// Word `at` (of query `query`, in group `group`) of up to MOST partial results, of which there are `count`, brought to one
// reference and one unit; word(c, i) reads word i of partial result c.
struct Merged {
  float m, e, l, a;  // the reference, the unit's exponent, the sum and the value
  __device__ __forceinline__ float average() const { return a / l * fast_exp2(e); }
};
template <typename L, uint32_t MOST, typename Word>
__device__ __forceinline__ Merged merge_parts(uint32_t count, uint32_t query, uint32_t group, uint32_t at, Word word) {
  float m[MOST], e[MOST];
  Merged r{kNoScore, -INFINITY, 0.f, 0.f};
#pragma unroll
  for (uint32_t c = 0; c < MOST; ++c) {
    m[c] = c < count ? word(c, L::kReferences + query) : kNoScore;
    e[c] = c < count ? word(c, L::kUnits + group * kQ4Queries + query) : float(kNoUnit);
    r.m = fmaxf(r.m, m[c]);
  }
#pragma unroll
  for (uint32_t c = 0; c < MOST; ++c) r.e = fmaxf(r.e, m[c] - r.m + e[c]);
#pragma unroll
  for (uint32_t c = 0; c < MOST; ++c) {
    if (c >= count) break;
    r.l = fmaf(word(c, L::kSums + query), fast_exp2(m[c] - r.m), r.l);
    r.a = fmaf(word(c, at), fast_exp2(m[c] - r.m + e[c] - r.e), r.a);
  }
  return r;
}

struct Q4Attention {
  const uint16_t* q;
  const uint8_t* cache;
  const int32_t* lengths;
  uint16_t* out;
  uint32_t ldq, heads, kv_heads, tiles;
  uint32_t share;   // query heads per key / value head
  int32_t length_offset;
  uint32_t blocks;  // groups of query heads per key / value head
  float* parts;     // split over more CTAs than a cluster holds: each leaves its partial result here
  uint32_t early;   // the grid is resident at once: the next kernel may start at entry
};

// CTAs of `warps` warps that an SM is to hold: 128 registers a thread for heads of 128, 96 for 64. Fewer warps with more
// registers, and more with fewer, are slower: 512 sequences of 64 query heads over 8 and 576 positions 47.4 us at 20 warps an
// SM, 48.3 at 16, 49.2 at 24; 256 of 32 over 8 heads of 128 and 1152 positions 70.2 at 16, 74.8 at 12, 89.9 at 20. CTAs of eight
// warps come in two kinds, two to an SM as long as that holds the grid (192 pairs of 60 tiles 6.8 us against 7.7, 256 grouped
// pairs of 72 9.0 against 11.5, when this was set), else three (384 pairs of 72 10.6 against 11.5, heads of 64 only: those of
// 128 do not fit three, and two rounds of two are still faster, 384 pairs of 72 20.3 us against 21.6 by CTAs of four warps).
constexpr uint32_t q4_resident(int head, int warps) { return head == 128 ? 16 / warps : warps == 8 ? 2 : 20 / warps; }

template <int G, int RP, int WARPS, int RESIDENT>
__global__ void __launch_bounds__(32 * WARPS, RESIDENT) decode_attention_q4_kernel(Q4Attention p) {
  using L = Q4Smem<G, WARPS>;
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr uint32_t kWidth = 64 * G, kTileBytes = G * kQ4Block, kPieceTiles = kQ4Piece / kTileBytes;
  constexpr uint32_t CP = q4_columns(RP), TP = q4_tiles_at_once(G, RP);
  const uint32_t warp = warp_id(), lane = lane_id(), g = lane >> 2, t = lane & 3u;
  const uint32_t chunks = gridDim.x, chunk = blockIdx.x, s = blockIdx.z;
  // (Integer divisions by numbers only known at launch cost about 25 instructions each: none where there is nothing to
  // divide.)
  const uint32_t share = RP == 1 ? 1 : p.share, kvh = p.blocks == 1 ? blockIdx.y : blockIdx.y / p.blocks;
  const uint32_t first = (blockIdx.y - kvh * p.blocks) * RP;  // of the key / value head's query heads
  const uint32_t queries = min(uint32_t(RP), share - first);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBarrierOffset) + warp * kRing;
  uint8_t* ring = smem + warp * L::kWarpRing;
  if (lane == 0) {
#pragma unroll
    for (uint32_t i = 0; i < kRing; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
  if (p.early) pdl_launch_dependents();
  pdl_wait();

  const int64_t want = int64_t(p.lengths[s]) + p.length_offset;
  const uint32_t capacity = p.tiles * kQ4Tile;
  const uint32_t len = want <= 0 ? 0u : want < int64_t(capacity) ? uint32_t(want) : capacity;
  // The CTA's tiles [t_begin, t_end), a run of them for each warp.
  const uint32_t used = (len + kQ4Tile - 1) / kQ4Tile, per = chunks == 1 ? used : (used + chunks - 1) / chunks;
  const uint32_t t_begin = min(used, chunk * per), t_end = min(used, t_begin + per);
  const uint32_t share_w = (t_end - t_begin + WARPS - 1) / WARPS;
  const uint32_t w_begin = min(t_end, t_begin + warp * share_w), w_end = min(t_end, w_begin + share_w);
  const uint32_t pieces = (w_end - w_begin + kPieceTiles - 1) / kPieceTiles;
  const uint8_t* base = p.cache + (size_t(s) * p.kv_heads + kvh) * p.tiles * kTileBytes;
  auto fetch = [&](uint32_t piece, uint32_t slot) {
    const uint32_t tile = w_begin + piece * kPieceTiles, bytes = min(kPieceTiles, w_end - tile) * kTileBytes;
    mbar_arrive_expect_tx(&full[slot], bytes);
    bulk_load(ring + slot * kQ4Piece, base + size_t(tile) * kTileBytes, bytes, &full[slot]);
  };
  if (lane == 0) {
#pragma unroll
    for (uint32_t i = 0; i < kRing; ++i)
      if (i < pieces) fetch(i, i);
  }

  // The query fragments: lane (g, t) holds dimensions 16 t .. 16 t + 15 of each group of its column's query, the group scaled
  // by a power of two to a greatest magnitude below 2.
  uint32_t qf[G][8];
  float qs[G][2], unit[G][2];
#pragma unroll
  for (int i = 0; i < G; ++i) {
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (g % CP < queries) {
      const uint4* q4 = reinterpret_cast<const uint4*>(
          p.q + size_t(s) * p.ldq + size_t(kvh * share + first + g % CP) * kWidth + i * 64 + t * 16);
      a = q4[0];
      b = q4[1];
    }
    float x[16], lo[8], hi[8], greatest = 0.f;
    unpack8(a, lo);
    unpack8(b, hi);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      x[d] = lo[d];
      x[8 + d] = hi[d];
      greatest = fmax3(greatest, fabsf(lo[d]), fabsf(hi[d]));
    }
    greatest = fmaxf(greatest, __shfl_xor_sync(0xFFFFFFFFu, greatest, 1));
    greatest = fmaxf(greatest, __shfl_xor_sync(0xFFFFFFFFu, greatest, 2));
    const uint32_t exponent = min(max(__float_as_uint(greatest) >> 23, 1u), 253u);
    const float down = __uint_as_float((254u - exponent) << 23), up = kDecodeLog2e * __uint_as_float(exponent << 23);
    unit[i][0] = __shfl_sync(0xFFFFFFFFu, up, 8 * t);  // of the lane's own columns, 2 t and 2 t + 1
    unit[i][1] = __shfl_sync(0xFFFFFFFFu, up, 8 * t + 4);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      // pair0 and pair1 of a word and of its swapped form give dimensions n and n + 4 of a word's eight
      const int d = n / 4 * 8 + n % 4;
      const __half2 h = __floats2half2_rn(x[d] * down, x[d + 4] * down);
      qf[i][n] = *reinterpret_cast<const uint32_t*>(&h);
      sum += __low2float(h) + __high2float(h);
    }
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
    sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
    qs[i][0] = __shfl_sync(0xFFFFFFFFu, sum, 8 * t);
    qs[i][1] = __shfl_sync(0xFFFFFFFFu, sum, 8 * t + 4);
  }

  Q4State<G> st;
  st.m[0] = st.m[1] = kNoScore;
  st.l[0] = st.l[1] = 0.f;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    st.inv[i][0] = st.inv[i][1] = inverse_unit(kNoUnit);
    st.low[i][0] = st.low[i][1] = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) st.acc[i][n][c] = 0.f;
  }
  const Q4Constants kc{in_register(0x00F000F0u), in_register(16u)};
  uint32_t slot = 0, phase = 0, limit = pieces;
  bool ok = true;
  for (uint32_t piece = 0; piece < limit; ++piece) {
    const bool landed = mbar_wait(&full[slot], phase, kWatchFull, nullptr);
    if (ok && !__all_sync(0xFFFFFFFFu, landed)) {
      // A copy that does not land: nothing more is issued, and the copies in flight are each waited for, bounded.
      ok = false;
      limit = min(limit, piece + kRing);
    }
    if (ok) {
      const uint32_t tile = w_begin + piece * kPieceTiles, end = min(tile + kPieceTiles, w_end);
      const uint32_t left = min(len, end * kQ4Tile) - tile * kQ4Tile;  // positions of this piece
      const uint8_t* data = ring + slot * kQ4Piece;
      if (left == kPieceTiles * kQ4Tile) {
#pragma unroll
        for (uint32_t i = 0; i < kPieceTiles; i += TP)
          q4_tiles<G, RP, true>(st, qf, qs, unit, data + i * kTileBytes, TP * kQ4Tile, g, t, kc);
      } else {
#pragma unroll 1
        for (uint32_t i = 0; i * kQ4Tile < left; i += TP)
          q4_tiles<G, RP, false>(st, qf, qs, unit, data + i * kTileBytes, left - i * kQ4Tile, g, t, kc);
      }
      __syncwarp();
      if (lane == 0 && piece + kRing < pieces) fetch(piece + kRing, slot);
    }
    if (++slot == kRing) {
      slot = 0;
      phase ^= 1u;
    }
  }
  if (!p.early) pdl_launch_dependents();

  // The warp's partial result, (values in the unit, reference, unit, sum) of each query, into its own ring: the columns of
  // one query (CP / 2 lanes apart) and the lanes' sums come together first.
  __syncwarp();
  float* part = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int c = 0; c < (RP > 1 ? 2 : 1); ++c) {
    float m = st.m[c];
#pragma unroll
    for (int o = CP / 2; o < 4; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    float l = st.l[c] * fast_exp2(st.m[c] - m);
#pragma unroll
    for (int o = CP / 2; o < 32; o <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, o);
    const uint32_t query = 2 * t % CP + c;
    const bool writes = 2 * t < CP && query < queries;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const float own = st.m[c] - m + float(unit_exponent(st.inv[i][c]));
      float e = own;
#pragma unroll
      for (int o = CP / 2; o < 4; o <<= 1) e = fmaxf(e, __shfl_xor_sync(0xFFFFFFFFu, e, o));
      const float f = fast_exp2(own - e);
      if (g == 0 && writes) part[L::kUnits + i * kQ4Queries + query] = e;
      float rest = st.low[i][c] * f;
#pragma unroll
      for (int o = CP / 2; o < 32; o <<= 1) rest += __shfl_xor_sync(0xFFFFFFFFu, rest, o);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        float lo = st.acc[i][n][c] * (f * kCodeOne), hi = st.acc[i][n][2 + c] * (f * kCodeOne);
#pragma unroll
        for (int o = CP / 2; o < 4; o <<= 1) {
          lo += __shfl_xor_sync(0xFFFFFFFFu, lo, o);
          hi += __shfl_xor_sync(0xFFFFFFFFu, hi, o);
        }
        if (writes) {
          part[query * L::kStride + i * 64 + 8 * n + g] = lo + rest;
          part[query * L::kStride + i * 64 + 8 * (4 + n) + g] = hi + rest;
        }
      }
    }
    if (g == 0 && writes) {
      part[L::kReferences + query] = m;
      part[L::kSums + query] = l;
    }
  }
  __syncthreads();
  // The warps' results together: output, or the CTA's own partial result, in its shared memory or in the workspace.
  const bool whole = chunks == 1 && p.parts == nullptr;
  float* merge = p.parts != nullptr
                     ? p.parts + (size_t(s * gridDim.y + blockIdx.y) * chunks + chunk) * (L::kPart / 4)
                     : reinterpret_cast<float*>(smem + L::kMergeOffset);
  uint16_t* out = p.out + (size_t(s) * p.heads + kvh * share + first) * kWidth;
  for (uint32_t i = threadIdx.x; i < queries * kWidth; i += 32 * WARPS) {
    const uint32_t query = i / kWidth, at = query * L::kStride + i % kWidth;
    const uint32_t group = i % kWidth / 64;
    const Merged r = merge_parts<L, WARPS>(WARPS, query, group, at, [&](uint32_t w, uint32_t i) {
      return reinterpret_cast<const float*>(smem + w * L::kWarpRing)[i];
    });
    if (whole) {
      out[query * kWidth + q4_dimension(i % kWidth)] = float_to_bf16(len == 0 ? 0.f : r.average());
    } else {
      merge[at] = r.a;
      if (i % 64 == 0) merge[L::kUnits + group * kQ4Queries + query] = r.e;
      if (i % kWidth == 0) {
        merge[L::kReferences + query] = r.m;
        merge[L::kSums + query] = r.l;
      }
    }
  }
  if (whole || p.parts != nullptr) return;
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  // Each CTA finishes its share of the outputs, reading every CTA's partial result.
  for (uint32_t i = chunk * 32 * WARPS + threadIdx.x; i < queries * kWidth; i += chunks * 32 * WARPS) {
    const uint32_t query = i / kWidth, at = query * L::kStride + i % kWidth;
    const Merged r = merge_parts<L, kQ4MaxChunks>(chunks, query, i % kWidth / 64, at,
                                                  [&](uint32_t c, uint32_t i) { return ld_cluster(merge + i, c); });
    out[query * kWidth + q4_dimension(i % kWidth)] = float_to_bf16(len == 0 ? 0.f : r.average());
  }
  // No CTA leaves while another may still read its shared memory.
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// One CTA per (sequence, query head): the partial results of `chunks` CTAs, summed in a fixed order. kMergeThreads / 64 G
// threads share a dimension, and each has kMergeBatch values on their way at once, the first of them while the references
// are compared. (A loop that loaded the last few of them one after the other cost up to 2 us.)
constexpr uint32_t kMergeThreads = 512, kMergeBatch = 8;
static_assert(kQ4MaxSplits <= kMergeThreads, "a thread for each partial result");

template <int G>
__global__ void __launch_bounds__(kMergeThreads) decode_merge_q4_kernel(Q4Attention p, uint32_t chunks, uint32_t rp) {
  using L = Q4Smem<G, 4>;
  constexpr uint32_t kWidth = 64 * G, kShares = kMergeThreads / kWidth, kPart = L::kPart / 4;
  constexpr uint32_t kFactors = (kQ4MaxSplits + kMergeBatch * kShares - 1) / (kMergeBatch * kShares) * (kMergeBatch * kShares);
  __shared__ float factor[G][kFactors];
  __shared__ float warp_greatest[1 + G][kMergeThreads / 32], warp_l[kMergeThreads / 32];
  __shared__ float sums[kShares][kWidth];
  pdl_wait();
  pdl_launch_dependents();
  const uint32_t share = p.share, h = blockIdx.x, s = blockIdx.y;
  const uint32_t kvh = h / share, block = h % share / rp, query = h % share % rp;
  const float* parts = p.parts + size_t((s * p.kv_heads + kvh) * p.blocks + block) * chunks * kPart;
  const uint32_t at = threadIdx.x % kWidth, part = threadIdx.x / kWidth;
  const float* values = parts + query * L::kStride + at;
  float v[kMergeBatch];
  auto load = [&](uint32_t from) {
#pragma unroll
    for (uint32_t i = 0; i < kMergeBatch; ++i) {
      const uint32_t c = from + part + i * kShares;
      v[i] = c < chunks ? values[c * kPart] : 0.f;
    }
  };
  load(0);
  const bool has = threadIdx.x < chunks;
  const float m = has ? parts[threadIdx.x * kPart + L::kReferences + query] : kNoScore;
  float e[G];
#pragma unroll
  for (int i = 0; i < G; ++i)
    e[i] = has ? parts[threadIdx.x * kPart + L::kUnits + i * kQ4Queries + query] : float(kNoUnit);
  const float part_l = has ? parts[threadIdx.x * kPart + L::kSums + query] : 0.f;
  float (*of_warps)[kMergeThreads / 32] = warp_greatest;
  auto greatest = [&](auto& x) {  // of every thread, for each of x
    constexpr int kCount = sizeof(x) / sizeof(float);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x[i] = fmaxf(x[i], __shfl_xor_sync(0xFFFFFFFFu, x[i], o));
      if (lane_id() == 0) of_warps[i][warp_id()] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kCount; ++i)
#pragma unroll
      for (uint32_t w = 0; w < (kQ4MaxSplits + 31) / 32; ++w) x[i] = fmaxf(x[i], of_warps[i][w]);  // (the others have none)
    of_warps += kCount;
  };
  float reference[1] = {m}, unit[G];
  greatest(reference);
  const float below = m - reference[0], l_warp = warp_sum(part_l * fast_exp2(below));
#pragma unroll
  for (int i = 0; i < G; ++i) unit[i] = below + e[i];
  greatest(unit);
#pragma unroll
  for (int i = 0; i < G; ++i)
    if (threadIdx.x < kFactors) factor[i][threadIdx.x] = has ? fast_exp2(below + e[i] - unit[i]) : 0.f;
  if (lane_id() == 0) warp_l[warp_id()] = l_warp;
  __syncthreads();
  float a = 0.f;
  for (uint32_t from = 0; from < chunks; from += kMergeBatch * kShares) {
    if (from > 0) load(from);
#pragma unroll
    for (uint32_t i = 0; i < kMergeBatch; ++i) a = fmaf(v[i], factor[at / 64][from + part + i * kShares], a);
  }
  sums[part][at] = a;
  __syncthreads();
  if (threadIdx.x >= kWidth) return;
  float l = 0.f;
#pragma unroll
  for (uint32_t w = 0; w < kMergeThreads / 32; ++w) l += warp_l[w];
  a = 0.f;
#pragma unroll
  for (uint32_t i = 0; i < kShares; ++i) a += sums[i][at];
  const bool empty = int64_t(p.lengths[s]) + p.length_offset <= 0;
  const Merged all{0.f, at < 64 ? unit[0] : unit[G - 1], l, a};
  p.out[(size_t(s) * p.heads + h) * kWidth + q4_dimension(at)] = float_to_bf16(empty ? 0.f : all.average());
}

// How the positions of a pair (a sequence's key / value head and block of query heads) are shared out: CTAs of `warps`
// warps, `chunks` of them to a pair, merged through a cluster's shared memory or, with `parts`, through the workspace.
struct Q4Split {
  uint32_t warps, chunks;
  bool parts;
};

// Up to twice as many CTAs as fit the GPU (lengths differ, and a second round fills what the short ones leave), as long as
// each has 12 tiles, and more where there are many pairs, whose CTAs hide one another's latency. Measured on a B200 over 726
// grids of up to 768 pairs and four times as many, of 4 to 4096 tiles, at full and at ragged lengths, against CTAs of two, four
// and eight warps, clusters of two to eight and up to 148 CTAs through the workspace: 3 % behind the best of these on average,
// 39 % at worst (440 ragged pairs of 24 tiles of heads of 128, which two rounds of eight-warp CTAs serve in 12.5 us and one of
// four-warp CTAs in 9.0). us (w warps, c CTAs, p through the workspace): 768 pairs of 72 w4c1 15.4, w8c1 17.4, w4c2 18.8; 192
// of 72 w8c1 7.4, w4c1 8.8, w4c2 9.2, w4c4 10.5; 96 of 256 w4c8 12.3, w4c1 14.8; 16 of 1024 (128-wide) 15.5, w4c37p 16.4,
// w4c16p 17.8, w4c8 21.9; 16 of 4096 (128-wide) w4c37p 36.9, w4c64p 39.0, w4c16p 48.3, w4c8 73. Four times 768 of 72: w2c1 45.5,
// w4c1 48.3 (a CTA's latency weighs more than its width there).
Q4Split q4_split(uint64_t pairs, uint32_t tiles, uint32_t head) {
  const uint64_t sms = uint64_t(sm_count());
  const uint64_t chunks = std::min(2 * q4_resident(head, 4) * sms / pairs, tiles * sms / (12 * sms + 32 * pairs));
  if (chunks < 3) return Q4Split{pairs >= 20 * sms ? 2u : pairs <= 3 * sms && tiles >= 16 ? 8u : 4u, 1, false};
  if (chunks <= 12) return Q4Split{4, chunks < 6 ? 4u : 8u, false};
  // As many as fit at once, or twice that, whichever has its rounds of CTAs done first: whole pieces to each warp, and a
  // CTA's fixed cost about that of 12 tiles.
  const uint64_t slots = q4_resident(head, 4) * sms;
  uint64_t least = UINT64_MAX;
  uint32_t best = 0;
  for (uint32_t rounds = 1; rounds <= 2; ++rounds) {
    const uint32_t most = uint32_t(std::min<uint64_t>({chunks, kQ4MaxSplits, rounds * slots / pairs}));
    const uint32_t per = ((tiles + most - 1) / most + 15) / 16 * 16, count = (tiles + per - 1) / per;
    const uint64_t cost = (pairs * count + slots - 1) / slots * (per + 12);
    if (cost < least) {
      least = cost;
      best = count;
    }
  }
  return Q4Split{4, best, true};
}

template <int G, int RP, int WARPS, int RESIDENT = q4_resident(64 * G, WARPS)>
tempo_status launch_attention_warps(const Q4Attention& base, uint32_t seqs, uint32_t chunks, cudaStream_t stream) {
  Q4Attention p = base;
  auto kernel = decode_attention_q4_kernel<G, RP, WARPS, RESIDENT>;
  const bool cluster = chunks > 1 && p.parts == nullptr;
  const tempo_status status = set_smem(reinterpret_cast<const void*>(kernel), Q4Smem<G, WARPS>::kBytes);
  if (status != TEMPO_OK) return status;
  p.early = single_wave(uint64_t(p.kv_heads) * p.blocks * seqs * chunks, 16 / WARPS);
  return launch(kernel, dim3(chunks, p.kv_heads * p.blocks, seqs), dim3(32 * WARPS),
                Q4Smem<G, WARPS>::kBytes, stream, cluster ? chunks : 1, "decode_attention_q4_kernel", p);
}

template <int G, int RP>
tempo_status launch_attention(const Q4Attention& base, uint32_t seqs, const Q4Split& split, float* workspace,
                              cudaStream_t stream) {
  Q4Attention p = base;
  p.parts = split.parts ? workspace : nullptr;
  if (split.warps == 2) return launch_attention_warps<G, RP, 2>(p, seqs, split.chunks, stream);
  if (split.warps == 8) {
    const uint64_t pairs = uint64_t(p.kv_heads) * p.blocks * seqs;
    if (G == 1 && pairs > q4_resident(64, 8) * uint64_t(sm_count()))
      return launch_attention_warps<G, RP, 8, G == 1 ? 3 : 2>(p, seqs, split.chunks, stream);
    return launch_attention_warps<G, RP, 8>(p, seqs, split.chunks, stream);
  }
  tempo_status status = launch_attention_warps<G, RP, 4>(p, seqs, split.chunks, stream);
  if (status != TEMPO_OK || !split.parts) return status;
  return launch(decode_merge_q4_kernel<G>, dim3(p.heads, seqs), dim3(kMergeThreads), 0, stream, 1, "decode_merge_q4_kernel", p,
                split.chunks, uint32_t(RP));
}

// Query heads of one CTA: all that share a key / value head, up to eight.
uint32_t q4_queries(uint32_t head, uint32_t share) {
  return share == 1 ? 1 : share == 2 && head == 64 ? 2 : share <= 4 ? 4 : 8;
}

uint64_t q4_workspace(uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head, uint32_t capacity) {
  const uint32_t share = heads / kv_heads, rp = q4_queries(head, share);
  const uint64_t pairs = uint64_t(seqs) * kv_heads * ((share + rp - 1) / rp);
  const Q4Split split = q4_split(pairs, capacity / kQ4Tile, head);
  return split.parts ? pairs * split.chunks * (head == 64 ? Q4Smem<1, 4>::kPart : Q4Smem<2, 4>::kPart) : 0;
}

tempo_status check_attention(const char* what, uint32_t seqs, uint32_t heads, uint32_t kv_heads) {
  if (heads == 0 || heads % kv_heads || seqs > 65535 || heads > 65535)
    return fail(TEMPO_ERR_VALUE, "%s: seqs %u (up to 65535), heads %u must be a multiple of kv_heads %u (both up to "
                "65535)", what, seqs, heads, kv_heads);
  return TEMPO_OK;
}

// What the three entry points check alike; `what` names the call.
tempo_status check_cache(const char* what, const void* cache, uint32_t seqs, uint32_t kv_heads, uint32_t head,
                         uint32_t capacity) {
  if (seqs == 0 || kv_heads == 0 || kv_heads > 65535 || capacity == 0 || capacity % kQ4Tile ||
      (head != 64 && head != 128))
    return fail(TEMPO_ERR_VALUE, "%s: seqs %u kv_heads %u (up to 65535) head %u (64 or 128) capacity %u (a multiple of "
                "16)", what, seqs, kv_heads, head, capacity);
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
  if (rows == 0 || rows > 0x7FFFFFFFu || width > ldq || ldq % 8)
    return fail(TEMPO_ERR_VALUE, "tempo_kv_store_q4: rows %u, row stride %u (a multiple of 8, at least %llu)", rows, ldq,
                static_cast<unsigned long long>(width));
  if (qkv == nullptr || !aligned16(qkv) || seq_of == nullptr || pos_of == nullptr)
    return fail(TEMPO_ERR_VALUE, "tempo_kv_store_q4: 16-byte aligned rows, a sequence and a position of each are needed");
  Q4Rows p{};
  p.rows = const_cast<uint16_t*>(static_cast<const uint16_t*>(qkv)) + size_t(heads) * head;
  p.cache = static_cast<uint8_t*>(cache);
  p.seq_of = seq_of;
  p.pos_of = pos_of;
  p.ld = ldq;
  p.seqs = seqs;
  p.kv_heads = kv_heads;
  p.tiles = capacity / kQ4Tile;
  auto kernel = wide_rows(p) ? (head == 64 ? kv_store_q4_kernel<1, true> : kv_store_q4_kernel<2, true>)
                             : (head == 64 ? kv_store_q4_kernel<1, false> : kv_store_q4_kernel<2, false>);
  return launch_rows(kernel, p, rows, head / kQ4Group, static_cast<cudaStream_t>(stream), "kv_store_q4_kernel");
}

extern "C" tempo_status tempo_kv_load_q4(const void* cache, void* kv, uint32_t ldo, const int32_t* seq_of,
                                         const int32_t* pos_of, uint32_t rows, uint32_t seqs, uint32_t kv_heads,
                                         uint32_t head, uint32_t capacity, void* stream) {
  tempo_status status = check_cache("tempo_kv_load_q4", cache, seqs, kv_heads, head, capacity);
  if (status != TEMPO_OK) return status;
  const uint64_t width = 2ull * kv_heads * head;
  if (rows == 0 || rows > 0x7FFFFFFFu || width > ldo || ldo % 8)
    return fail(TEMPO_ERR_VALUE, "tempo_kv_load_q4: rows %u, row stride %u (a multiple of 8, at least %llu)", rows, ldo,
                static_cast<unsigned long long>(width));
  if (kv == nullptr || !aligned16(kv) || seq_of == nullptr || pos_of == nullptr)
    return fail(TEMPO_ERR_VALUE, "tempo_kv_load_q4: a 16-byte aligned output, a sequence and a position of each row are "
                "needed");
  Q4Rows p{};
  p.rows = static_cast<uint16_t*>(kv);
  p.cache = const_cast<uint8_t*>(static_cast<const uint8_t*>(cache));
  p.seq_of = seq_of;
  p.pos_of = pos_of;
  p.ld = ldo;
  p.seqs = seqs;
  p.kv_heads = kv_heads;
  p.tiles = capacity / kQ4Tile;
  auto kernel = wide_rows(p) ? (head == 64 ? kv_load_q4_kernel<1, true> : kv_load_q4_kernel<2, true>)
                             : (head == 64 ? kv_load_q4_kernel<1, false> : kv_load_q4_kernel<2, false>);
  return launch_rows(kernel, p, rows, head / kQ4Group, static_cast<cudaStream_t>(stream), "kv_load_q4_kernel");
}

extern "C" tempo_status tempo_decode_attention_q4_workspace(uint32_t seqs, uint32_t heads, uint32_t kv_heads,
                                                            uint32_t head, uint32_t capacity, uint64_t* bytes) {
  alignas(16) static const char placeholder[16] = {};
  tempo_status status = check_cache("tempo_decode_attention_q4_workspace", placeholder, seqs, kv_heads, head, capacity);
  if (status != TEMPO_OK) return status;
  status = check_attention("tempo_decode_attention_q4_workspace", seqs, heads, kv_heads);
  if (status != TEMPO_OK) return status;
  if (bytes == nullptr) return fail(TEMPO_ERR_VALUE, "tempo_decode_attention_q4_workspace: nowhere to put the size");
  *bytes = q4_workspace(seqs, heads, kv_heads, head, capacity);
  return TEMPO_OK;
}

extern "C" tempo_status tempo_decode_attention_q4(const void* q, uint32_t ldq, const void* cache,
                                                  const int32_t* lengths, int32_t length_offset, void* out,
                                                  uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t head,
                                                  uint32_t capacity, void* workspace, uint64_t workspace_bytes,
                                                  void* stream) {
  tempo_status status = check_cache("tempo_decode_attention_q4", cache, seqs, kv_heads, head, capacity);
  if (status != TEMPO_OK) return status;
  status = check_attention("tempo_decode_attention_q4", seqs, heads, kv_heads);
  if (status != TEMPO_OK) return status;
  if (uint64_t(heads) * head > ldq || ldq % 8)
    return fail(TEMPO_ERR_VALUE, "tempo_decode_attention_q4: the query row stride %u must be a multiple of 8 and at "
                "least %llu", ldq, static_cast<unsigned long long>(uint64_t(heads) * head));
  if (q == nullptr || !aligned16(q) || out == nullptr || !aligned16(out) || lengths == nullptr)
    return fail(TEMPO_ERR_VALUE, "tempo_decode_attention_q4: 16-byte aligned queries and output and the lengths are "
                "needed");
  const uint64_t needed = q4_workspace(seqs, heads, kv_heads, head, capacity);
  if (needed > 0 && (workspace == nullptr || !aligned16(workspace) || workspace_bytes < needed))
    return fail(TEMPO_ERR_VALUE, "tempo_decode_attention_q4: a 16-byte aligned workspace of %llu bytes is needed, got "
                "%llu", static_cast<unsigned long long>(needed), static_cast<unsigned long long>(workspace_bytes));
  const uint32_t share = heads / kv_heads, rp = q4_queries(head, share);
  Q4Attention p{};
  p.q = static_cast<const uint16_t*>(q);
  p.cache = static_cast<const uint8_t*>(cache);
  p.lengths = lengths;
  p.out = static_cast<uint16_t*>(out);
  p.ldq = ldq;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.share = share;
  p.tiles = capacity / kQ4Tile;
  p.length_offset = length_offset;
  p.blocks = (share + rp - 1) / rp;
  const Q4Split split = q4_split(uint64_t(seqs) * kv_heads * p.blocks, p.tiles, head);
  float* parts = static_cast<float*>(workspace);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head == 128) {
    if (rp == 1) return launch_attention<2, 1>(p, seqs, split, parts, st);
    return rp == 4 ? launch_attention<2, 4>(p, seqs, split, parts, st) : launch_attention<2, 8>(p, seqs, split, parts, st);
  }
  if (rp == 1) return launch_attention<1, 1>(p, seqs, split, parts, st);
  if (rp == 2) return launch_attention<1, 2>(p, seqs, split, parts, st);
  return rp == 4 ? launch_attention<1, 4>(p, seqs, split, parts, st) : launch_attention<1, 8>(p, seqs, split, parts, st);
}
