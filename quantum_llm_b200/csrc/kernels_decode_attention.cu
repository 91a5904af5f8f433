// Attention of one new token per sequence over the paged cache, for a batch of sequences of
// different lengths (qllm_k_decode_attention), and the attention weight that each cached key received.
//
//   z_t = scale * q . K_t,  p_t = exp(z_t) / sum_u exp(z_u),  out = sum_t p_t V_t
//   weights_out_t = weights_in_t + sum over the group's query heads of p_t
//
// HBM-bound: a key costs 2 * 2 D bytes (F16; 2 (D + 2) Q8, 2 (D / 2 + 2) Q4H) and 4 D operations per query
// head of its group, at most 16 operations a byte for a group of eight.
//
// Work split.  An item is (sequence, head set): up to eight query heads of one kv head, or of `heads`
// neighbouring kv heads (Q8, below).  The units of 64 tokens of all items stand in one line, and block b of C
// takes the share [b W / C, (b + 1) W / C) of it, whatever the lengths are: one wave of equal blocks for one
// long sequence and for a ragged batch alike.  A block finishes an item that lies inside its share by itself;
// of one that does not it leaves (maximum, sum, unnormalised output) in the workspace -- at most one item that
// began before its share and one that goes on after it, hence two places per block -- and a second launch
// joins those.  The split depends on the lengths alone, so the bits of a result do not depend on scheduling.
//
// Inner product on the tensor cores (mma.sync, FP32 out; operands below) with the CACHE as the M operand:
// S^T = K q^T has 16 keys x 8 heads, out^T = V^T P^T 16 dims x 8 heads, so that a group of up to eight query
// heads fills the N = 8 side instead of a sixteenth to a half of an M side.  tcgen05 wants an M of 64 or 128
// and its operands in shared memory; here the keys go from global memory straight into the registers of a
// fragment (no shared memory, no barrier) because the order of k inside a product is free: a lane takes
// whichever 16 bytes of a row it can load at once, and the query is laid out to match.  For V^T of Q8 and Q4H
// the pairs of keys that a fragment packs are put together by byte permutes.  Key 2 r stands in row r of a 16-key
// block, key 2 r + 1 in row r + 8, so that a lane's two keys (scales, scores) are neighbours.
//
// Numerics.  Codes of Q8 and Q4H records are small integers: K's meet the query as INT8 (mma.sync m16n8k32), the query as a
// 23-bit integer (24-bit with FP32 rows) relative to the largest of its row in three digits of base 256, so that every product and sum
// of a digit is exact (one INT8 instruction takes the time of an F16 one of half as many dimensions, and K needs no
// conversion); V's are exact in F16.  The records' scales multiply scores and weights in FP32.  For an F16 cache the query is
// scaled by a power of two to [2^8, 2^9) and becomes F16: exact for F16 and (down to 2^-22 of the largest) BF16 rows, two terms
// (22 bits) for FP32 rows.  The weights p that meet V are two terms of 11 bits with FP32 and F16 rows, and one with BF16 rows: off by
// 2^-11 of each weight at most there, an eighth of the output's own rounding.  Over an F16 cache the terms are TF32 (m16n8k8, F16 values
// are TF32 values), which holds a weight of any size to that many bits: the keys that make up the output may all be far below
// the largest weight, where that key's V is near zero (F16 terms: 20 nats below, FP32 rows were off by 0.7 to 1 %, 40 nats
// below by all; the time of two TF32 terms is 1 to 7 % above that of F16 terms, of one 0 to 1 %).  Over Q8 and Q4H the terms are
// F16, of p times V's scale: the reference is set so that the largest of those is 2^7 and moved when one would exceed 2^15 (one vote per tile instead
// of a reduction), F16 holds them down to 2^-32 of the largest, and a key whose V is small has a small scale.
//
// Measured on one B200 (copy 6554 GB/s), device time of both launches: 64 sequences of up to 8192 tokens, F16, 32 query and 4 kv
// heads of 128, BF16 rows: 102 us, 6.1 TB/s of cache, HBM-bound; 7 of up to 20001, F16, 16 heads of 64, FP32 rows, with weights:
// 58 us, 4.1 TB/s (two terms a query and a weight: instruction issue, then the weights' pass); 96 of up to 4500, Q8, 40 and 8 heads
// of 128, F16 rows, with weights: 136 us, 3.6 TB/s, after a pause (unpacking bytes: instruction issue) and 143 to 154 us in calls one after
// the other; 1 of 32768, Q4H, 40 and 8 heads of 128: 21 us, 1.6 TB/s (a block's share is some 150 tokens a warp: set-up, merge and join
// are more than half); 1 of 1000, F16: 9.7 us (latency alone).
#include <type_traits>

#include "kernels.h"
#include "kv_batch.cuh"
#include "launch.cuh"

namespace qllm {

namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kUnit = 64;          // tokens
constexpr uint32_t kItemBytes = 96U * 1024U;  // what a block could read in the time an item costs it beside its tokens
constexpr uint32_t kMaxBlocks = 768;    // of the first launch; places in the workspace
constexpr uint32_t kHeads = 8;          // query heads of an item per kv head
constexpr uint32_t kWeightTokens = 4 * kThreads;
constexpr size_t kSharedByDefault = 47U * 1024U;  // of a launch without asking for more, beside the static arrays
// log2: the largest p of a warp stands between 2^kLift (when the reference was set) and 2^kTop < 65504
constexpr float kLift = 7.0F, kTop = 15.0F;
constexpr float kLog2e = 1.4426950408889634F;

// kv heads that share a block.  A Q8 record is 2 bytes longer than a multiple of 32, so neighbouring heads'
// records share sectors: four warps on four heads of the same tokens fetch them once.
__host__ __device__ inline uint32_t head_set(const KvBatch& c) {
  if (c.encoding != QLLM_KV_Q8) return 1U;
  return c.kv_heads % 4U == 0U ? 4U : c.kv_heads % 2U == 0U ? 2U : 1U;
}

struct Plan {
  uint32_t heads;          // kv heads of an item
  uint32_t group, tiles;   // query heads per kv head, and tiles of eight of them
  uint32_t items;          // per sequence
  uint32_t cost;           // of an item beside its tokens, in units
  uint32_t rows;           // of one place: heads * 8
  size_t place;            // floats of one place: [rows] maxima, [rows] sums, [rows][head_dim] outputs
  float* partials;         // [kMaxBlocks][2][place]
  uint2* spans;            // [sequences * items]: first and last block of an item
  float* lse;              // [sequences, q_heads], log2 (weights only)
  float* scores;           // [sequences, q_heads, capacity], log2 (weights only)
  size_t bytes;
};
inline size_t up16(size_t n) { return (n + 15U) & ~static_cast<size_t>(15U); }
Plan plan_of(const KvBatch& c, uint32_t q_heads, bool weights, void* workspace) {
  Plan p{};
  p.heads = head_set(c);
  p.group = q_heads / c.kv_heads;
  p.tiles = (p.group + kHeads - 1U) / kHeads;
  p.items = c.kv_heads / p.heads * p.tiles;
  const size_t unit = kUnit * p.heads * kv_layer_bytes(c.encoding, 1U, 1U, c.head_dim);
  p.cost = static_cast<uint32_t>((kItemBytes + unit - 1U) / unit);
  p.rows = p.heads * kHeads;
  p.place = static_cast<size_t>(p.rows) * (2U + c.head_dim);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  size_t n = 0;
  const auto take = [&](size_t bytes) {
    uint8_t* p0 = at ? at + n : nullptr;
    n += up16(bytes);
    return p0;
  };
  p.partials = reinterpret_cast<float*>(take(kMaxBlocks * 2U * p.place * sizeof(float)));
  p.spans = reinterpret_cast<uint2*>(take(static_cast<size_t>(c.sequences) * p.items * sizeof(uint2)));
  if (weights) {
    const size_t rows = static_cast<size_t>(c.sequences) * q_heads;
    p.lse = reinterpret_cast<float*>(take(rows * sizeof(float)));
    p.scores = reinterpret_cast<float*>(take(rows * kv_capacity(c) * sizeof(float)));
  }
  p.bytes = n;
  return p;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void add_scaled(float4& to, const float4& x, float f) {
  to.x = fmaf(x.x, f, to.x);
  to.y = fmaf(x.y, f, to.y);
  to.z = fmaf(x.z, f, to.z);
  to.w = fmaf(x.w, f, to.w);
}
// out / sum to four elements of a row; zeros where no key counts, whatever its values are (0 times infinity is none).
template <typename T>
__device__ __forceinline__ void put_four(T* to, const float4& out, float sum) {
  const bool none = sum == 0.0F;
  const float scale = 1.0F / sum;
  put_row(to, none ? 0.0F : out.x * scale);
  put_row(to + 1, none ? 0.0F : out.y * scale);
  put_row(to + 2, none ? 0.0F : out.z * scale);
  put_row(to + 3, none ? 0.0F : out.w * scale);
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma1688(float (&d)[4], float a0, float a1, float a2, float a3, uint32_t b0, uint32_t b1) {  // TF32
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t to_tf32(float v) {
  uint32_t d;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(d) : "f"(v));
  return d;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <uint32_t kMask, uint32_t kFlip>
__device__ __forceinline__ uint32_t mask_flip(uint32_t v) {  // (v & mask) ^ flip
  return (v & kMask) ^ kFlip;
}
__device__ __forceinline__ uint32_t half2_sub(uint32_t v, uint32_t c) {
  uint32_t d;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(d) : "r"(v), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t half2_fma(uint32_t v, uint32_t m, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(v), "r"(m), "r"(c));
  return d;
}
// Cache records are read once: past L1.
template <int kWords>
__device__ __forceinline__ void load_words(uint32_t* d, const uint8_t* p) {
  if constexpr (kWords == 4)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "l"(p));
  else if constexpr (kWords == 2)
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "l"(p));
  else
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(d[0]) : "l"(p));
}

// Shared memory by its 32-bit address, the offset in the instruction.
template <int kOffset>
__device__ __forceinline__ uint32_t shared_word(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1+%2];" : "=r"(v) : "r"(at), "n"(kOffset) : "memory");
  return v;
}
template <int kOffset>
__device__ __forceinline__ float shared_half(uint32_t at) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1+%2];" : "=h"(v) : "r"(at), "n"(kOffset) : "memory");
  return __half2float(__ushort_as_half(v));
}
template <int kStep, int kN, int kI = 0>
__device__ __forceinline__ void shared_words(uint32_t at, uint32_t (&w)[kN]) {
  w[kI] = shared_word<kStep * kI>(at);
  if constexpr (kI + 1 < kN) shared_words<kStep, kN, kI + 1>(at, w);
}

// Four nibbles (two's complement) at bits 0, 4, 8, 12 of each 16-bit half -> pairs of F16, one per nibble position:
// 0x6400 | (n ^ 8) is 1024 + n + 8, and with the nibble four bits higher 1024 + 16 (n + 8).
__device__ __forceinline__ void nibbles_to_half(uint32_t w, uint32_t (&h)[4]) {
  const uint32_t high = w >> 8U;
  h[0] = half2_sub(mask_flip<0x000F000FU, 0x64086408U>(w), 0x64086408U);
  h[1] = half2_fma(mask_flip<0x00F000F0U, 0x64806480U>(w), 0x2C002C00U, 0xD480D480U);      // / 16 - 72
  h[2] = half2_sub(mask_flip<0x000F000FU, 0x64086408U>(high), 0x64086408U);
  h[3] = half2_fma(mask_flip<0x00F000F0U, 0x64806480U>(high), 0x2C002C00U, 0xD480D480U);
}
// Signed bytes in bits 0-7 of each half -> F16: 0x6400 | (b ^ 0x80) is 1024 + b + 128.  (Left in, and the sum of the weights times
// 1152 taken off at the end, V's bias would cost FP32 sums four bits.)
__device__ __forceinline__ uint32_t bytes_to_half(uint32_t v) {
  return half2_sub(mask_flip<0x00FF00FFU, 0x64806480U>(v), 0x64806480U);
}

// ---- what depends on the encoding: how a lane's registers hold a 16-key block.
// lane = 4 r + c.  K: rows r (key 2 r) and r + 8 (key 2 r + 1).  V: keys 4 c .. 4 c + 3.
template <int ENC, int HD>
struct Layout {
  static constexpr bool kStaged = ENC == QLLM_KV_Q8;
  // blocks of 16 keys that a warp takes at a time: 16 - 64 registers of K and of V (Q4H, HD 128: 4 blocks spill, 31 us
  // against 25 us with 2 for one sequence of 32768; F16, HD 64: 2 blocks leave room for three blocks of threads to a
  // multiprocessor instead of four, 64 us against 57 us for 7 sequences of up to 20001)
  static constexpr int kBlocks = ENC == QLLM_KV_Q4H ? 2 : 1;
  static constexpr int kRegs = ENC == QLLM_KV_F16 ? HD / 4 : ENC == QLLM_KV_Q4H ? HD / 16 : 1;  // of K, and of V, per block
  static constexpr int kKWords = ENC == QLLM_KV_Q4H ? (HD % 128 == 0 ? 4 : 2) : 4;      // words per load
  static constexpr int kVWords = ENC == QLLM_KV_Q4H ? (HD == 128 ? 2 : HD == 256 ? 4 : 1) : 4;
  // staged rows: the 16-byte windows that cover a record wherever it begins
  static constexpr int kWindows = HD / 16 + 1;
  static constexpr int kPitch = 16 * kWindows;
  static constexpr int kStage = 2 * 16 * kPitch;
  static constexpr int kStages = HD == 64 ? 4 : HD <= 192 ? 3 : 2;  // as many as leave room for kBlocksPerSm

  // K meets the query as F16 (steps of 16 dimensions) or, where its codes are integers, as INT8 (steps of 32)
  static constexpr bool kIntegerKeys = ENC != QLLM_KV_F16;
  static constexpr int kSteps = kIntegerKeys ? HD / 32 : HD / 16;
  static constexpr int kPerRegister = kIntegerKeys ? 4 : 2;
  // dimension of part `part` of fragment register b (0, 1) in step `step`, lane c.  `turn`: 2 if the words of a Q8 row
  // begin two codes before the record does (words(), below).
  static __device__ __forceinline__ uint32_t query_dim(int step, int b, int part, uint32_t c, uint32_t turn) {
    if constexpr (ENC == QLLM_KV_F16) return 8U * (c + 4U * (step / 2)) + 4U * (step % 2) + 2U * b + part;
    if constexpr (ENC == QLLM_KV_Q8) return turned(4U * (c + 4U * (2 * step + b)) + part, turn);
    const uint32_t word = (c + 4U * (step / kKWords)) * kKWords + step % kKWords;
    return 8U * word + 2U * part + b;
  }
  // first of the two neighbouring dimensions of output tile mt in lane r
  static __device__ __forceinline__ uint32_t out_dim(int mt, uint32_t r, uint32_t turn) {
    if constexpr (ENC == QLLM_KV_F16) return 8U * (r + 8U * (mt / 4)) + 2U * (mt % 4);
    if constexpr (ENC == QLLM_KV_Q8) return turned(4U * (r + 8U * (mt / 2)) + 2U * (mt % 2), turn);
    const uint32_t word = (r + 8U * (mt / 4 / kVWords)) * kVWords + (mt / 4) % kVWords;
    return 8U * word + 2U * (mt % 4);
  }
  static __device__ __forceinline__ uint32_t turned(uint32_t d, uint32_t turn) { return d < turn ? d + HD - turn : d - turn; }
};

// Where the keys of a 16-key block lie.
struct Block {
  const uint8_t* keys;   // K codes (values) of its first token and the warp's kv head; null: no page
  uint32_t place;        // of its first token in the page
  uint32_t count;        // keys that count, 0..16
};

// Walks every `step` tokens from `first` through the pages of a sequence, without a division after the start.
struct Cursor {
  uint32_t token, page, place;
  uint32_t step, step_pages, step_place;
  __device__ __forceinline__ Cursor(const KvBatch& c, uint32_t first, uint32_t step_) : token(first), step(step_) {
    page = first / c.page_tokens;
    place = first - page * c.page_tokens;
    step_pages = step / c.page_tokens;
    step_place = step - step_pages * c.page_tokens;
  }
  __device__ __forceinline__ void advance(const KvBatch& c) {
    token += step;
    page += step_pages;
    place += step_place;
    if (place >= c.page_tokens) {
      place -= c.page_tokens;
      ++page;
    }
  }
};

template <typename T, int ENC, int HD>
struct Traits {
  static constexpr bool kPrecise = sizeof(T) == 4;  // two F16 terms for the query,
  static constexpr bool kPreciseWeights = !std::is_same<T, __nv_bfloat16>::value;  // and for the weights
  // fragments of the query per step: F16 terms, or INT8 digits of an integer
  static constexpr int kTerms = Layout<ENC, HD>::kIntegerKeys ? 3 : kPrecise ? 2 : 1;
  static constexpr int kSteps = Layout<ENC, HD>::kSteps;
  static constexpr bool kQueryInRegisters = HD <= 128;
  static constexpr int kBlocksPerSm = HD == 64 ? 4 : HD == 128 ? 3 : 2;
  // the queries of one kv head: rows 16 bytes apart from a multiple of 128 (free of bank conflicts), then fragments in their place
  static constexpr int kQueryPitch = HD * static_cast<int>(sizeof(T)) + 16;
  static constexpr size_t kRowsBytes = static_cast<size_t>(kHeads) * kQueryPitch;
  // Fragments go through shared memory where four warps share them and each makes a quarter, and where they stay there.
  static constexpr bool kSharedQuery = !Layout<ENC, HD>::kStaged;
  static constexpr size_t kFragmentBytes = kSharedQuery || !kQueryInRegisters ? static_cast<size_t>(kSteps) * 32 * kTerms * sizeof(uint2) : 0;
  static constexpr size_t kQueryBytes = kSharedQuery ? kRowsBytes + kFragmentBytes : kRowsBytes > kFragmentBytes ? kRowsBytes : kFragmentBytes;
  static constexpr int kRow = HD + 4;  // floats of one head in the merge area
  static constexpr size_t kMergeBytes = (kWarps * kHeads * kRow + 2 * kWarps * kHeads) * sizeof(float);
  static constexpr size_t kRingBytes = Layout<ENC, HD>::kStaged ? static_cast<size_t>(kWarps) * Layout<ENC, HD>::kStages * Layout<ENC, HD>::kStage : 0;
  static constexpr size_t kShared = (kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes) + kQueryBytes * (ENC == QLLM_KV_Q8 ? 4 : 1);
};

// Largest magnitude, as the bits of a float, of a row that four lanes share (c = 0 .. 3); NaN counts as the largest.
template <int HD, typename T>
__device__ __forceinline__ uint32_t row_maximum(const T* row, uint32_t c) {
  const uint4* from = reinterpret_cast<const uint4*>(row) + c;
  uint32_t top = 0U;
#pragma unroll
  for (int i = 0; i < HD * static_cast<int>(sizeof(T)) / 64; ++i) {
    const uint4 x = from[4 * i];
    const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (uint32_t v : word) {
      if constexpr (sizeof(T) == 4)
        top = max(top, v & 0x7FFFFFFFU);
      else
        top = __vmaxu2(top, v & 0x7FFF7FFFU);
    }
  }
  if constexpr (sizeof(T) == 2) {
    const unsigned short half = static_cast<unsigned short>(max(top & 0xFFFFU, top >> 16U));
    if constexpr (std::is_same<T, __half>::value) top = __float_as_uint(__half2float(__ushort_as_half(half)));
    else top = static_cast<uint32_t>(half) << 16U;
    top &= 0x7FFFFFFFU;
  }
  top = max(top, __shfl_xor_sync(0xffffffffU, top, 1));
  return max(top, __shfl_xor_sync(0xffffffffU, top, 2));
}
__device__ __forceinline__ int exponent(float x) {  // of a positive number: x in [2^exponent, 2^(exponent + 1))
  const bool small = x < 0x1p-126F;
  return static_cast<int>(__float_as_uint(small ? x * 0x1p24F : x) >> 23U) - (small ? 151 : 127);
}
__device__ __forceinline__ float power_of_two(int n) { return __int_as_float((n + 127) << 23); }  // n in [-126, 127]
// For operands that fit 32 bits most of the time.
__device__ __forceinline__ unsigned long long divide(unsigned long long a, uint32_t b) {
  return a >> 32U ? a / b : static_cast<uint32_t>(a) / b;
}

// State of the online softmax and of the output in one warp: heads 2 c and 2 c + 1 of the lane.
template <int HD>
struct Running {
  float out[HD / 16][4];   // out^T tiles: dims (d, heads 2c, 2c+1), (d + 1, the same)
  float reference[2];      // log2
  float sum[2];            // of the lane's own keys
};

// Scores of one tile (kN blocks) -> weights; moves the reference where a score calls for it.
// s[b] = {key 2r: heads 2c, 2c+1; key 2r+1: the same}, log2 units, masked keys -inf.  vscale: of keys 2r, 2r+1.
template <int HD, int kN, bool kScaled>
__device__ __forceinline__ void softmax_tile(Running<HD>& run, float (&s)[kN][4], const float (&vscale)[kN][2]) {
  float bias[kN][2];
#pragma unroll
  for (int b = 0; b < kN; ++b)
#pragma unroll
    for (int k = 0; k < 2; ++k)  // a scale that is infinite or NaN makes the output so, not the reference
      bias[b][k] = kScaled ? __log2f(fminf(fmaxf(fabsf(vscale[b][k]), 0x1p-24F), 65504.0F)) : 0.0F;
  float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int b = 0; b < kN; ++b)
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) top[h] = fmaxf(top[h], s[b][2 * k + h] + bias[b][k]);
  if (__any_sync(0xffffffffU, top[0] > run.reference[0] + kTop || top[1] > run.reference[1] + kTop)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffU, top[h], o));
      const float next = fmaxf(run.reference[h], top[h] - kLift);
      const float factor = run.reference[h] == -INFINITY ? 0.0F : exp2_fast(run.reference[h] - next);
      run.reference[h] = next;
      run.sum[h] *= factor;
#pragma unroll
      for (int mt = 0; mt < HD / 16; ++mt) {
        run.out[mt][h] *= factor;
        run.out[mt][2 + h] *= factor;
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float reference = run.reference[h] == -INFINITY ? 0.0F : run.reference[h];
#pragma unroll
    for (int b = 0; b < kN; ++b)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float p = exp2_fast(s[b][2 * k + h] - reference);
        run.sum[h] += p;
        s[b][2 * k + h] = kScaled ? p * vscale[b][k] : p;
      }
  }
}

// Weights of a block as the B operand (keys x heads) of an F16 product, one or two terms.
template <bool kPrecise>
__device__ __forceinline__ void weight_fragments(const float (&p)[4], uint32_t (&hi)[2], uint32_t (&lo)[2]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t h = pack_half(p[2 * k], p[2 * k + 1]);
    hi[k] = transpose8(h);
    if constexpr (kPrecise) {
      const float2 f = unpack_half(h);
      lo[k] = transpose8(pack_half(p[2 * k] - f.x, p[2 * k + 1] - f.y));
    }
  }
}

// Weights of a block as the B operands of two TF32 products (keys 4c, 4c + 1 and 4c + 2, 4c + 3), one or two terms each.  The
// two halves of the FP32 words are transposed one after the other.
template <bool kPrecise>
__device__ __forceinline__ void weight_fragments_tf32(const float (&p)[4], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t x = __float_as_uint(p[2 * k]), y = __float_as_uint(p[2 * k + 1]);
    const uint32_t low = transpose8(__byte_perm(x, y, 0x5410)), high = transpose8(__byte_perm(x, y, 0x7632));
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // key 4c + 2i + k
      const float w = __uint_as_float(__byte_perm(low, high, i ? 0x7632U : 0x5410U));
      hi[2 * i + k] = to_tf32(w);
      if constexpr (kPrecise) lo[2 * i + k] = to_tf32(w - __uint_as_float(hi[2 * i + k]));
    }
  }
}

__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from, bool there) {
  const uint32_t bytes = there ? 16U : 0U;  // 0: the 16 bytes become zero and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
template <int kOffset>
__device__ __forceinline__ void copy16_if(bool wanted, uint32_t to, const uint8_t* from) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\t@p cp.async.cg.shared.global [%0+%3], [%1], 16;\n\t}" ::"r"(to), "l"(from),
               "r"(static_cast<uint32_t>(wanted)), "n"(kOffset) : "memory");
}

__device__ __forceinline__ Block take_block(const Block& mine, int lane) {
  Block b;
  b.keys = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffU, reinterpret_cast<unsigned long long>(mine.keys), lane));
  b.place = __shfl_sync(0xffffffffU, mine.place, lane);
  b.count = __shfl_sync(0xffffffffU, mine.count, lane);
  return b;
}

template <typename T, int ENC, int HD>
struct Warp {
  using L = Layout<ENC, HD>;
  using X = Traits<T, ENC, HD>;
  static constexpr int kN = L::kBlocks;
  const DecodeAttentionArgs& a;
  uint32_t lane, r, c;
  uint32_t kv_head, sequence;
  const uint2* fragments;  // of the query heads, in shared memory: [step][term][lane]
  float scale[2];          // of heads 2c, 2c+1: score units -> log2
  Running<HD> run;

  __device__ __forceinline__ uint2 query(const uint2 (&regs)[X::kQueryInRegisters ? X::kSteps * X::kTerms : 1], int step, int term) const {
    if constexpr (X::kQueryInRegisters) return regs[step * X::kTerms + term];
    return fragments[(step * X::kTerms + term) * 32 + lane];
  }

  // Offsets inside a page's layer are below 2^32 (checked by the host).
  uint32_t stride;       // bytes from a token's record to the next token's (of one head)
  uint32_t to_values;    // from K records to V records
  uint32_t records;      // of K in a page
  __device__ __forceinline__ void layout() {
    records = a.cache.page_tokens * a.cache.kv_heads;
    stride = ENC == QLLM_KV_F16 ? a.cache.kv_heads * HD * 2U : ENC == QLLM_KV_Q8 ? a.cache.kv_heads * (HD + 2U) : HD / 2U;
    to_values = records * (ENC == QLLM_KV_F16 ? HD * 2U : ENC == QLLM_KV_Q8 ? HD + 2U : HD / 2U + 2U);
  }
  __device__ __forceinline__ Block block_at(const Cursor& at, uint32_t last) const {
    Block b{nullptr, at.place, 0U};
    if (at.token < last) {
      const uint8_t* layer = kv_page(a.cache, sequence, at.page);
      if (layer) {
        const uint32_t offset = ENC == QLLM_KV_F16   ? at.place * stride + kv_head * (HD * 2U)
                                : ENC == QLLM_KV_Q8 ? at.place * stride + kv_head * (HD + 2U)
                                                     : (kv_head * a.cache.page_tokens + at.place) * stride;
        b.keys = layer + offset;
        b.count = min(16U, last - at.token);
      }
    }
    return b;
  }
  // Q4H: the scales of a block's keys
  __device__ __forceinline__ const uint8_t* scales_of(const Block& b) const {
    const uint32_t record = kv_head * a.cache.page_tokens + b.place;
    return b.keys + (records * (HD / 2U) - record * (HD / 2U) + record * 2U);
  }

  // ---- registers (F16, Q4H)
  __device__ __forceinline__ void load_keys(const Block& b, uint32_t (&k)[L::kRegs], uint32_t& scales) {
    if (b.count == 0U) {
#pragma unroll
      for (int i = 0; i < L::kRegs; ++i) k[i] = 0U;
      scales = 0U;
      return;
    }
    const uint8_t* p = b.keys + 2U * r * stride + (ENC == QLLM_KV_F16 ? 16U : 4U * L::kKWords) * c;
    if constexpr (ENC == QLLM_KV_F16) {
#pragma unroll
      for (int row = 0; row < 2; ++row)
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) load_words<4>(&k[row * (HD / 8) + 4 * j], p + row * stride + 64 * j);
    } else {
#pragma unroll
      for (int row = 0; row < 2; ++row)
#pragma unroll
        for (int j = 0; j < HD / 32 / L::kKWords; ++j)
          load_words<L::kKWords>(&k[row * (HD / 32) + L::kKWords * j], p + row * (HD / 2) + 16 * L::kKWords * j);
      load_words<1>(&scales, scales_of(b) + 4U * r);
    }
  }
  __device__ __forceinline__ void load_values(const Block& b, uint32_t (&v)[L::kRegs], uint32_t& scales) {
    const uint8_t* p = b.keys + to_values + 4U * c * stride + (ENC == QLLM_KV_F16 ? 16U : 4U * L::kVWords) * r;
    constexpr int kWordsOnce = L::kVWords, kLoads = HD * (ENC == QLLM_KV_F16 ? 4 : 1) / 64 / kWordsOnce;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool there = 4U * c + q < b.count;
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        uint32_t* d = &v[(q * kLoads + j) * kWordsOnce];
#pragma unroll
        for (int i = 0; i < kWordsOnce; ++i) d[i] = 0U;
        if (there) load_words<kWordsOnce>(d, p + q * stride + 32 * kWordsOnce * j);
      }
    }
    scales = 0U;
    if constexpr (ENC == QLLM_KV_Q4H) {
      if (b.count) load_words<1>(&scales, scales_of(b) + to_values + 4U * r);
    }
  }
  // The three digits' products (each exact) as one FP32 score.
  static __device__ __forceinline__ void join_digits(const int (&d)[3][4], float (&s)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      s[i] = fmaf(static_cast<float>(d[2][i]), 65536.0F, fmaf(static_cast<float>(d[1][i]), 256.0F, static_cast<float>(d[0][i])));
  }
  template <int kQ>
  __device__ __forceinline__ void score(const uint2 (&q)[kQ], const uint32_t (&k)[L::kRegs], float (&s)[4]) const {
    if constexpr (ENC == QLLM_KV_F16) {
      // The tensor cores cut their FP32 sums off instead of rounding them: with FP32 rows no more than 64 dimensions go into
      // one, and the low terms have one of their own (relative error of the output at head_dim 256 and 20000 keys: 2.8e-6
      // with one sum, 0.6e-6 so).
      constexpr int kChain = X::kPrecise ? 4 : X::kSteps;
      float low[4] = {};
      s[0] = s[1] = s[2] = s[3] = 0.0F;
#pragma unroll
      for (int from = 0; from < X::kSteps; from += kChain) {
        float high[4] = {};
#pragma unroll
        for (int step = from; step < from + kChain; ++step) {
          const int i = 2 * step;  // words 4 w, 4 w + 1 and 4 w + 2, 4 w + 3 of a chunk
#pragma unroll
          for (int term = 0; term < X::kTerms; ++term) {
            const uint2 f = query(q, step, term);
            mma16816(term == 0 ? high : low, k[i], k[HD / 8 + i], k[i + 1], k[HD / 8 + i + 1], f.x, f.y);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += high[i];
      }
      if constexpr (X::kTerms == 2) {  // of an infinite key the low terms have either sign
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] += fabsf(s[i]) == INFINITY ? 0.0F : low[i];
      }
    } else {
      // the even and the odd nibbles of a word as bytes, sixteen times their value
      int d[3][4] = {};
#pragma unroll
      for (int step = 0; step < X::kSteps; ++step) {
        const uint32_t k0 = k[step], k1 = k[HD / 32 + step];
#pragma unroll
        for (int digit = 0; digit < 3; ++digit) {
          const uint2 f = query(q, step, digit);
          mma16832(d[digit], (k0 << 4U) & 0xF0F0F0F0U, (k1 << 4U) & 0xF0F0F0F0U, k0 & 0xF0F0F0F0U, k1 & 0xF0F0F0F0U, f.x, f.y);
        }
      }
      join_digits(d, s);
    }
  }
  // One tile of V^T times the weights: a sum of its own, added by an instruction that rounds.  The tensor cores cut their FP32
  // sums off, and one that goes on over all keys of a warp drifts towards zero with their number (65536 keys, V of one sign, F16
  // rows: 96 to 99.9 % of the outputs were not the nearest F16 value, now 1 %; the additions cost 0 to 3 % of the time).
  static __device__ __forceinline__ void add_product(float (&out)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                     const uint32_t (&hi)[2], const uint32_t (&lo)[2]) {
    float tile[4] = {};
    if constexpr (X::kPreciseWeights) mma16816(tile, a0, a1, a2, a3, lo[0], lo[1]);
    mma16816(tile, a0, a1, a2, a3, hi[0], hi[1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] += tile[i];
  }
  // F16 cache: TF32 holds its values as they are, and weights of any size.
  __device__ __forceinline__ void add_values(const uint32_t (&v)[L::kRegs], const float (&p)[4]) {
    uint32_t hi[4], lo[4] = {};
    weight_fragments_tf32<X::kPreciseWeights>(p, hi, lo);
#pragma unroll
    for (int w = 0; w < HD / 64; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 f[4];  // dimensions d, d + 1 of keys 4c .. 4c + 3
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = unpack_half(v[(k * (HD / 64) + w) * 4 + i]);
        float tile[4] = {};
        if constexpr (X::kPreciseWeights) {
          mma1688(tile, f[0].x, f[0].y, f[1].x, f[1].y, lo[0], lo[1]);
          mma1688(tile, f[2].x, f[2].y, f[3].x, f[3].y, lo[2], lo[3]);
        }
        mma1688(tile, f[0].x, f[0].y, f[1].x, f[1].y, hi[0], hi[1]);
        mma1688(tile, f[2].x, f[2].y, f[3].x, f[3].y, hi[2], hi[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) run.out[4 * w + i][j] += tile[j];
      }
  }
  // Q4H: the blocks of a tile share one sum (one each: 1 x 32768 21.8 us instead of 21.3, 64 x 4500 with F16 rows 81.2 instead of 79.5).
  __device__ __forceinline__ void add_nibbles(const uint32_t (&v)[kN][L::kRegs], const float (&p)[kN][4]) {
    uint32_t hi[kN][2], lo[kN][2] = {};
#pragma unroll
    for (int b = 0; b < kN; ++b) weight_fragments<X::kPreciseWeights>(p[b], hi[b], lo[b]);
#pragma unroll
    for (int w = 0; w < HD / 64; ++w)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t selector = half ? 0x7632U : 0x5410U;
        float tile[2][4] = {};
#pragma unroll
        for (int b = 0; b < kN; ++b) {
          uint32_t even[4], odd[4];
          nibbles_to_half(__byte_perm(v[b][w], v[b][2 * (HD / 64) + w], selector), even);
          nibbles_to_half(__byte_perm(v[b][HD / 64 + w], v[b][3 * (HD / 64) + w], selector), odd);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if constexpr (X::kPreciseWeights) mma16816(tile[i], even[2 * i], even[2 * i + 1], odd[2 * i], odd[2 * i + 1], lo[b][0], lo[b][1]);
            mma16816(tile[i], even[2 * i], even[2 * i + 1], odd[2 * i], odd[2 * i + 1], hi[b][0], hi[b][1]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) run.out[4 * w + 2 * half + i][j] += tile[i][j];
      }
  }

  // ---- through shared memory (Q8): rows of windows, key 2r in row r, key 2r + 1 in row r + 8
  // The windows of the keys one after the other over the lanes: 144 bytes in a row of one key (four lanes to a key and
  // eight keys at a time need fewer instructions, but fetch a sector twice more often: 152 us against 144 us).
  static constexpr int kCopies = L::kStaged ? (16 * L::kWindows + 31) / 32 : 1;  // of a lane, for K and for V
  uint32_t key_at[kCopies];    // bytes from a block's first record to that of the lane's i-th window
  uint32_t row_at[kCopies];    // where the window goes in a stage
  uint32_t window_at[kCopies]; // 16 * window
  uint32_t key_shift[2], value_shift[4];  // of keys 2r, 2r + 1 and 4c .. 4c + 3: bytes from the block's first record, mod 16
  uint32_t turn_keys, turn_values;        // byte selectors that put the tail in the place of a turned row's first two bytes
  __device__ __forceinline__ void layout_staged() {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const uint32_t index = lane + 32U * i, key = index / L::kWindows, window = index % L::kWindows;
      key_at[i] = key * stride;
      row_at[i] = (key / 2U + 8U * (key & 1U)) * L::kPitch + 16U * window;
      window_at[i] = 16U * window;
    }
#pragma unroll
    for (uint32_t k = 0; k < 2U; ++k) key_shift[k] = (2U * r + k) * stride & 15U;
#pragma unroll
    for (uint32_t k = 0; k < 4U; ++k) value_shift[k] = (4U * c + k) * stride & 15U;
  }
  __device__ __forceinline__ void stage(const Block& b, uint32_t to) {
    if (b.count == 16U) {
      const uintptr_t base = reinterpret_cast<uintptr_t>(b.keys) & ~static_cast<uintptr_t>(15U);
      const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(b.keys)) & 15U;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const uint8_t* from = reinterpret_cast<const uint8_t*>(base) + (((shift + key_at[i]) & ~15U) + window_at[i]);
        const bool wanted = i + 1 < kCopies || 16 * L::kWindows % 32 == 0 || lane < 16U * L::kWindows % 32U;
        copy16_if<0>(wanted, to + row_at[i], from);
        copy16_if<16 * L::kPitch>(wanted, to + row_at[i], from + to_values);  // V begins on 16 bytes
      }
      return;
    }
    // keys that do not count become zeros, and their address only has to be one that exists
    const uint8_t* base = b.keys ? b.keys : reinterpret_cast<const uint8_t*>(a.cache.page_tables);
    const uint32_t step = b.keys ? stride : 0U, to_v = b.keys ? to_values : 0U;
    for (uint32_t index = lane; index < 16U * L::kWindows; index += 32U) {
      const uint32_t key = index / L::kWindows, window = index % L::kWindows;
      const uint8_t* from =
          reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(base + key * step) & ~static_cast<uintptr_t>(15U)) + 16U * window;
      const uint32_t row = to + (key / 2U + 8U * (key & 1U)) * L::kPitch + 16U * window;
      copy16(row, from, key < b.count);
      copy16(row + 16U * L::kPitch, from + to_v, key < b.count);
    }
  }
  // What is left to know of a staged block: keys that count, and where its first record begins in its row.
  static __device__ __forceinline__ uint32_t staged_as(const Block& b) {
    return b.count << 4U | (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(b.keys)) & 15U);
  }

  // The warp's part of tokens [first, last) of the sequence: every `phases`-th block of 16 from `phase` on.  begin() starts
  // the first loads, which need no query; tokens() does the rest.
  struct Start {
    uint32_t k[L::kStaged ? 1 : kN][L::kRegs], v[L::kStaged ? 1 : kN][L::kRegs], kscale[L::kStaged ? 1 : kN], vscale[L::kStaged ? 1 : kN];
    Block now[L::kStaged ? 1 : kN];
    uint32_t staged[L::kStages - 1];  // of the tiles on their way
    Block ahead;
    uint32_t tiles;
  };
  __device__ __forceinline__ void begin(Start& x, Cursor& at, uint32_t first, uint32_t last, uint32_t phase, uint32_t phases, uint32_t ring) {
    const uint32_t blocks = (last - first + 15U) / 16U;
    const uint32_t mine = blocks > phase ? (blocks - phase + phases - 1U) / phases : 0U;
    x.tiles = (mine + kN - 1U) / kN;
    if constexpr (!L::kStaged) {
      const Block b0 = block_at(at, last);
      at.advance(a.cache);
#pragma unroll
      for (int b = 0; b < kN; ++b) {
        x.now[b] = take_block(b0, b);
        load_keys(x.now[b], x.k[b], x.kscale[b]);
      }
#pragma unroll
      for (int b = 0; b < kN; ++b) load_values(x.now[b], x.v[b], x.vscale[b]);
    } else {
#pragma unroll
      for (int i = 0; i < L::kStages - 1; ++i) {
        const Block b = block_at(at, last);
        at.advance(a.cache);
        x.staged[i] = staged_as(b);
        if (static_cast<uint32_t>(i) < x.tiles) stage(b, ring + i * L::kStage);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
    }
    x.ahead = block_at(at, last);
    at.advance(a.cache);
  }
  template <int kQ>
  __device__ __forceinline__ void tokens(Start& x, Cursor& at, const uint2 (&q)[kQ], uint32_t first, uint32_t last, uint32_t phase, uint32_t phases,
                                         float* scores, size_t capacity, uint32_t heads_here, uint32_t ring) {
    if constexpr (!L::kStaged) {
      for (uint32_t tile = 0; tile < x.tiles; ++tile) {
        float s[kN][4], vs[kN][2];
        uint32_t count[kN];
#pragma unroll
        for (int b = 0; b < kN; ++b) {
          score(q, x.k[b], s[b]);
          count[b] = x.now[b].count;
          if constexpr (ENC == QLLM_KV_Q4H) {
            const float2 ks = unpack_half(x.kscale[b]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              s[b][h] *= ks.x * scale[h];
              s[b][2 + h] *= ks.y * scale[h];
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              s[b][h] *= scale[h];
              s[b][2 + h] *= scale[h];
            }
          }
          if (count[b] < 16U) {
#pragma unroll
            for (uint32_t k = 0; k < 2U; ++k)
              if (2U * r + k >= count[b]) s[b][2 * k] = s[b][2 * k + 1] = -INFINITY;
          }
          if (scores) put_scores(scores, capacity, heads_here, first + 16U * (phase + phases * (tile * kN + b)), last, s[b]);
        }
        const bool more = tile + 1U < x.tiles;
        if (more) {
#pragma unroll
          for (int b = 0; b < kN; ++b) {
            x.now[b] = take_block(x.ahead, b);
            load_keys(x.now[b], x.k[b], x.kscale[b]);
          }
        }
#pragma unroll
        for (int b = 0; b < kN; ++b) {
          const float2 f = ENC == QLLM_KV_Q4H ? unpack_half(x.vscale[b]) : make_float2(1.0F, 1.0F);
          vs[b][0] = f.x;
          vs[b][1] = f.y;
          if (count[b] < 16U) {
            if (2U * r >= count[b]) vs[b][0] = 0.0F;
            if (2U * r + 1U >= count[b]) vs[b][1] = 0.0F;
          }
        }
        softmax_tile<HD, kN, ENC != QLLM_KV_F16>(run, s, vs);
#pragma unroll
        for (int b = 0; b < kN; ++b)
          if constexpr (ENC == QLLM_KV_F16) add_values(x.v[b], s[b]);
        if constexpr (ENC == QLLM_KV_Q4H) add_nibbles(x.v, s);
        if (more) {
#pragma unroll
          for (int b = 0; b < kN; ++b) load_values(x.now[b], x.v[b], x.vscale[b]);
          x.ahead = block_at(at, last);
          at.advance(a.cache);
        }
      }
    } else if (a.cache.kv_heads & 1U) {
      staged_tokens<true>(x, at, q, first, last, phase, phases, scores, capacity, heads_here, ring);
    } else {
      staged_tokens<false>(x, at, q, first, last, phase, phases, scores, capacity, heads_here, ring);
    }
  }
  template <bool kAlternate, int kQ>
  __device__ __forceinline__ void staged_tokens(Start& x, Cursor& at, const uint2 (&q)[kQ], uint32_t first, uint32_t last, uint32_t phase,
                                                uint32_t phases, float* scores, size_t capacity, uint32_t heads_here, uint32_t ring) {
    // not unrolled over the stages: the loop is some 450 instructions, and three copies of it waited for instructions
    uint32_t here = ring, there = ring + (L::kStages - 1) * L::kStage;  // of this tile, and of the one staged next
#pragma unroll 1
    for (uint32_t tile = 0; tile < x.tiles; ++tile) {
      asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 2) : "memory");
      __syncwarp();  // everybody's copies have arrived, and the tile before has been read
      const uint32_t staged = x.staged[0];
#pragma unroll
      for (int i = 0; i + 2 < L::kStages; ++i) x.staged[i] = x.staged[i + 1];
      x.staged[L::kStages - 2] = staged_as(x.ahead);
      if (tile + L::kStages - 1U < x.tiles) stage(x.ahead, there);
      asm volatile("cp.async.commit_group;" ::: "memory");
      x.ahead = block_at(at, last);
      at.advance(a.cache);
      staged_block<kAlternate>(q, staged, here, first + 16U * (phase + phases * tile), last, scores, capacity, heads_here);
      there = here;
      here = here + L::kStage == ring + L::kStages * L::kStage ? ring : here + L::kStage;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  // `token`: of the block's first key; the scores of keys that lie on no page are -inf and belong there too
  __device__ __forceinline__ void put_scores(float* scores, size_t capacity, uint32_t heads_here, uint32_t token, uint32_t last,
                                             const float (&s)[4]) const {
    float* to = scores + 2U * c * capacity + token + 2U * r;
    if (token + 16U <= last) {  // rows of scores hold a multiple of 16, blocks begin at one
      if (2U * c < heads_here) *reinterpret_cast<float2*>(to) = make_float2(s[0], s[2]);
      if (2U * c + 1U < heads_here) *reinterpret_cast<float2*>(to + capacity) = make_float2(s[1], s[3]);
      return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (2U * c + h >= heads_here) continue;
      if (token + 2U * r < last) to[h * capacity] = s[h];
      if (token + 2U * r + 1U < last) to[h * capacity + 1U] = s[2 + h];
    }
  }
  // The codes of a staged record in words, word x + kLanes * i for lane x of the kLanes that share the row.  A record begins on
  // a 2-byte boundary, and the words are those of memory: where the first holds the two bytes before the record, the one
  // behind the last full word (`tail`) has the last two codes.  Those take the place of the first two bytes (`selector`): the
  // lane then holds the dimensions turned round by two, the same for every key of a head when kv_heads is even.  When it is
  // odd, records begin one way and the other in turn, and the words of the odd ones are put together anew (`realign`).
  template <int kLanes, bool kAlternate, int kN2>
  __device__ __forceinline__ void words(uint32_t record, uint32_t x, bool realign, uint32_t selector, uint32_t (&w)[kN2], uint32_t& tail) const {
    constexpr int kApart = kLanes == 4 ? 1 : 4;  // lanes from x to x + 1
    const uint32_t from = record & ~3U;
    shared_words<4 * kLanes>(from + 4U * x, w);
    tail = shared_word<HD>(from);
    if constexpr (kAlternate) {
      if (!realign) return;
#pragma unroll
      for (int i = 0; i < kN2; ++i) {
        const uint32_t beside = __shfl_sync(0xffffffffU, w[i], lane + kApart);
        const uint32_t around = i + 1 < kN2 ? __shfl_sync(0xffffffffU, w[(i + 1) % kN2], lane - kApart * (kLanes - 1)) : tail;
        w[i] = __funnelshift_r(w[i], x + 1U < kLanes ? beside : around, 16U);
      }
    } else {
      w[0] = __byte_perm(w[0], tail, selector);
    }
  }
  template <bool kAlternate, int kQ>
  __device__ __forceinline__ void staged_block(const uint2 (&q)[kQ], uint32_t staged, uint32_t at, uint32_t token, uint32_t last,
                                               float* scores, size_t capacity, uint32_t heads_here) {
    const uint32_t count = staged >> 4U, shift = staged & 15U;
    float s[1][4], vs[1][2], ks[2];
    uint32_t w[2][HD / 16];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t row = at + (r + 8U * k) * L::kPitch + ((shift + key_shift[k]) & 15U);
      const bool odd = (kv_head + (kAlternate ? k : 0)) & 1U;
      uint32_t tail;
      words<4, kAlternate>(row, c, odd, turn_keys, w[k], tail);
      ks[k] = __half2float(__ushort_as_half(static_cast<unsigned short>(odd ? tail >> 16U : tail)));
      vs[0][k] = shared_half<16 * L::kPitch + HD>(row);
    }
    {
      int d[3][4] = {};
#pragma unroll
      for (int step = 0; step < X::kSteps; ++step)
#pragma unroll
        for (int digit = 0; digit < 3; ++digit) {
          const uint2 f = query(q, step, digit);
          mma16832(d[digit], w[0][2 * step], w[1][2 * step], w[0][2 * step + 1], w[1][2 * step + 1], f.x, f.y);
        }
      join_digits(d, s[0]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) s[0][2 * k + h] *= ks[k] * scale[h];
    if (count < 16U) {
#pragma unroll
      for (uint32_t k = 0; k < 2U; ++k)
        if (2U * r + k >= count) {
          s[0][2 * k] = s[0][2 * k + 1] = -INFINITY;
          vs[0][k] = 0.0F;
        }
    }
    if (scores) put_scores(scores, capacity, heads_here, token, last, s[0]);
    softmax_tile<HD, 1, true>(run, s, vs);
    uint32_t hi[2], lo[2] = {0U, 0U};
    weight_fragments<X::kPreciseWeights>(s[0], hi, lo);
    uint32_t v[4][HD / 32];
#pragma unroll
    for (uint32_t k = 0; k < 4U; ++k) {
      uint32_t tail;
      words<8, kAlternate>(at + (16U + 2U * c + k / 2U + 8U * (k & 1U)) * L::kPitch + ((shift + value_shift[k]) & 15U), r,
                           (kv_head + (kAlternate ? k : 0U)) & 1U, turn_values, v[k], tail);
    }
#pragma unroll
    for (int j = 0; j < HD / 32; ++j)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t selector = half ? 0x7632U : 0x5410U;
        const uint32_t even = __byte_perm(v[0][j], v[2][j], selector), odd = __byte_perm(v[1][j], v[3][j], selector);
        const uint32_t a0 = bytes_to_half(even), a1 = bytes_to_half(even >> 8U), a2 = bytes_to_half(odd), a3 = bytes_to_half(odd >> 8U);
        add_product(run.out[2 * j + half], a0, a1, a2, a3, hi, lo);
      }
  }
};

template <typename T, int ENC, int HD>
__global__ void __launch_bounds__(kThreads, Traits<T, ENC, HD>::kBlocksPerSm)
decode_attention_kernel(const __grid_constant__ DecodeAttentionArgs a, const __grid_constant__ Plan plan) {
  using X = Traits<T, ENC, HD>;
  using L = Layout<ENC, HD>;
  extern __shared__ __align__(16) uint8_t shared[];
  __shared__ unsigned long long warp_units[kWarps];
  __shared__ uint32_t start_sequence;
  __shared__ unsigned long long start_base;
  const uint32_t lane = threadIdx.x & 31U, warp = threadIdx.x >> 5U;
  const uint32_t capacity = kv_capacity(a.cache), sequences = a.cache.sequences;
  // of one item of a sequence: its cost stands before its tokens in the line; nothing for a sequence without tokens
  const auto units_of = [&](uint32_t s) {
    const uint32_t n = (min(a.lengths[s], capacity) + kUnit - 1U) / kUnit;
    return n ? n + plan.cost : 0U;
  };

  // ---- this block's share [begin, end) of the line of units
  const uint32_t per_thread = (sequences + kThreads - 1U) / kThreads;
  const uint32_t s0 = min(sequences, threadIdx.x * per_thread), s1 = min(sequences, s0 + per_thread);
  unsigned long long own = 0ULL;
  for (uint32_t s = s0; s < s1; ++s) own += units_of(s);
  own *= plan.items;
  unsigned long long upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(0xffffffffU, upto, o);
    if (lane >= static_cast<uint32_t>(o)) upto += t;
  }
  if (lane == 31U) warp_units[warp] = upto;
  __syncthreads();
  unsigned long long total = 0ULL, before = upto - own;
#pragma unroll
  for (uint32_t w = 0; w < kWarps; ++w) {
    if (w < warp) before += warp_units[w];
    total += warp_units[w];
  }
  const uint32_t blocks = static_cast<uint32_t>(min(static_cast<unsigned long long>(gridDim.x), total));
  if (blockIdx.x >= blocks) return;
  unsigned long long u = divide(blockIdx.x * total, blocks);
  const unsigned long long end = divide((blockIdx.x + 1ULL) * total, blocks);
  if (before <= u && u < before + own) {
    uint32_t s = s0;
    unsigned long long base = before;
    for (;; ++s) {
      const unsigned long long n = static_cast<unsigned long long>(units_of(s)) * plan.items;
      if (u < base + n) break;
      base += n;
    }
    start_sequence = s;
    start_base = base;
  }
  __syncthreads();
  uint32_t s = start_sequence;
  unsigned long long base = start_base;

  using W = Warp<T, ENC, HD>;
  W w{a};
  w.lane = lane;
  w.r = lane >> 2U;
  w.c = lane & 3U;
  w.layout();
  if constexpr (L::kStaged) w.layout_staged();
  const uint32_t in_set = warp % plan.heads, phase = warp / plan.heads, phases = kWarps / plan.heads;
  uint2* fragments = reinterpret_cast<uint2*>(shared + in_set * X::kQueryBytes + (X::kSharedQuery ? X::kRowsBytes : 0));
  uint8_t* area = shared + X::kQueryBytes * plan.heads;
  float* merge_max = reinterpret_cast<float*>(area);           // [warp][head]
  float* merge_sum = merge_max + kWarps * kHeads;
  float* merge_out = merge_sum + kWarps * kHeads;              // [warp][head][HD + 4]
  w.fragments = fragments;

  while (u < end) {
    const uint32_t length = min(a.lengths[s], capacity);
    const uint32_t n = length ? (length + kUnit - 1U) / kUnit + plan.cost : 0U;
    if (u >= base + static_cast<unsigned long long>(n) * plan.items) {
      base += static_cast<unsigned long long>(n) * plan.items;
      ++s;
      continue;
    }
    const uint32_t item = static_cast<uint32_t>(divide(u - base, n)), local = static_cast<uint32_t>(u - base - static_cast<unsigned long long>(item) * n);
    const uint32_t take = static_cast<uint32_t>(min(static_cast<unsigned long long>(n - local), end - u));
    const uint32_t from = max(local, plan.cost) - plan.cost, upto = max(local + take, plan.cost) - plan.cost;  // units of tokens
    if (from == upto) {  // the share ends before the item's first token
      u += take;
      continue;
    }
    const uint32_t first = from * kUnit, last = min(length, upto * kUnit);
    const uint32_t set = item / plan.tiles, tile = item % plan.tiles;
    const uint32_t heads_here = min(kHeads, plan.group - tile * kHeads);
    const uint32_t kv_head = set * plan.heads + in_set;
    const uint32_t head0 = kv_head * plan.group + tile * kHeads;  // first query head of this warp

    w.sequence = s;
    w.kv_head = kv_head;
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(area)) + warp * (L::kStages * L::kStage);
    const uint32_t turn = ENC == QLLM_KV_Q8 && !(a.cache.kv_heads & 1U) ? 2U * (kv_head & 1U) : 0U;  // see words()
    w.turn_keys = turn && w.c == 0U ? 0x3254U : 0x3210U;
    w.turn_values = turn && w.r == 0U ? 0x3254U : 0x3210U;
    Cursor at(a.cache, first + 16U * (phase + phases * (L::kStaged ? 0U : lane % W::kN)), 16U * phases * W::kN);
    typename W::Start x;
    __syncthreads();  // the merge area and the queries of the item before have been read
    // the query and (where it leaves room in the registers) the first keys are on their way together
    constexpr uint32_t kChunks = kHeads * HD * sizeof(T) / 16U, kRowChunks = HD * sizeof(T) / 16U;
    const uint32_t queries = static_cast<uint32_t>(__cvta_generic_to_shared(shared));
    for (uint32_t i = threadIdx.x; i < plan.heads * kChunks; i += kThreads) {
      const uint32_t h = i / kChunks, g = i % kChunks / kRowChunks, chunk = i % kRowChunks;
      const bool there = g < heads_here;
      const T* q = static_cast<const T*>(a.query) + static_cast<size_t>(s) * a.query_stride +
                   static_cast<size_t>((set * plan.heads + h) * plan.group + tile * kHeads + (there ? g : 0U)) * HD;
      copy16(queries + h * X::kQueryBytes + g * X::kQueryPitch + 16U * chunk, reinterpret_cast<const uint8_t*>(q) + 16U * chunk, there);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if constexpr (X::kQueryInRegisters) w.begin(x, at, first, last, phase, phases, ring);

    // ---- the query heads as fragments, scaled to [2^8, 2^9) or integers
    asm volatile("cp.async.wait_group %0;" ::"n"(X::kQueryInRegisters && L::kStaged ? L::kStages - 1 : 0) : "memory");
    __syncthreads();
    const T* row = reinterpret_cast<const T*>(shared + in_set * X::kQueryBytes + w.r * X::kQueryPitch);
    constexpr int kPer = L::kPerRegister;
    const uint32_t top_bits = row_maximum<HD>(row, w.c);
    const bool wrong = top_bits >= 0x7F800000U;  // a NaN or an infinity
    // F16: to [2^8, 2^9); INT8 digits: to [2^21, 2^22)
    const int up = top_bits != 0U && !wrong ? (L::kIntegerKeys ? 21 : 8) - exponent(__uint_as_float(top_bits)) : 0;
    const int down = -up - (ENC == QLLM_KV_Q4H ? 4 : 0);  // Q4H codes come times sixteen
    float unit = a.scale * kLog2e * power_of_two(down / 2) * power_of_two(down - down / 2);  // of head r
    if (L::kIntegerKeys && wrong) unit = NAN;  // integers would lose it
    // FP32 rows: stretched to the largest integer that three digits hold, one to two bits more
    float stretch = 1.0F;
    if constexpr (L::kIntegerKeys && X::kPrecise) {
      if (top_bits != 0U && !wrong) stretch = 127.0F * 65536.0F / (__uint_as_float(top_bits) * power_of_two(up / 2) * power_of_two(up - up / 2));
      unit /= stretch;
    }
    w.scale[0] = __shfl_sync(0xffffffffU, unit, 8U * w.c);
    w.scale[1] = __shfl_sync(0xffffffffU, unit, 8U * w.c + 4U);
    // two factors: one may not be a float by itself
    const float up0 = power_of_two(up / 2), up1 = power_of_two(up - up / 2);
    const auto make_terms = [&](int step, uint2 (&made)[3]) {
      uint32_t term[3][2] = {};
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float x[kPer];
#pragma unroll
        for (int part = 0; part < kPer; ++part) x[part] = row_value(row[L::query_dim(step, b, part, w.c, turn)]) * up0 * up1 * stretch;
        if constexpr (L::kIntegerKeys) {
#pragma unroll
          for (int part = 0; part < kPer; ++part) {
            // three digits of base 256, -128..127
            const int n = __float2int_rn(x[part]);
            const int d0 = static_cast<int8_t>(n), n1 = (n - d0) >> 8, d1 = static_cast<int8_t>(n1), d2 = (n1 - d1) >> 8;
            term[0][b] |= (static_cast<uint32_t>(d0) & 255U) << (8 * part);
            term[1][b] |= (static_cast<uint32_t>(d1) & 255U) << (8 * part);
            term[2][b] |= (static_cast<uint32_t>(d2) & 255U) << (8 * part);
          }
        } else {
          term[0][b] = pack_half(x[0], x[1]);
          const float2 f = unpack_half(term[0][b]);
          term[1][b] = pack_half(x[0] - f.x, x[1] - f.y);
        }
      }
#pragma unroll
      for (int i = 0; i < 3; ++i) made[i] = make_uint2(term[i][0], term[i][1]);
    };
    uint2 q[X::kQueryInRegisters ? X::kSteps * X::kTerms : 1];
    if constexpr (X::kSharedQuery) {
      for (int step = static_cast<int>(phase); step < X::kSteps; step += static_cast<int>(phases)) {
        uint2 made[3];
        make_terms(step, made);
#pragma unroll
        for (int i = 0; i < X::kTerms; ++i) fragments[(step * X::kTerms + i) * 32 + lane] = made[i];
      }
      __syncthreads();
      if constexpr (X::kQueryInRegisters) {
#pragma unroll
        for (int i = 0; i < X::kSteps * X::kTerms; ++i) q[i] = w.fragments[i * 32 + lane];
      }
    } else if constexpr (X::kQueryInRegisters) {
#pragma unroll
      for (int step = 0; step < X::kSteps; ++step) {
        uint2 made[3];
        make_terms(step, made);
#pragma unroll
        for (int i = 0; i < X::kTerms; ++i) q[step * X::kTerms + i] = made[i];
      }
    } else {  // the fragments take the queries' place
      uint2 made[X::kSteps][3];
#pragma unroll
      for (int step = 0; step < X::kSteps; ++step) make_terms(step, made[step]);
      __syncthreads();
      if (phase == 0U) {
#pragma unroll
        for (int step = 0; step < X::kSteps; ++step)
#pragma unroll
          for (int i = 0; i < X::kTerms; ++i) fragments[(step * X::kTerms + i) * 32 + lane] = made[step][i];
      }
      __syncthreads();
    }
    if constexpr (!X::kQueryInRegisters) w.begin(x, at, first, last, phase, phases, ring);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w.run.reference[h] = -INFINITY;
      w.run.sum[h] = 0.0F;
#pragma unroll
      for (int mt = 0; mt < HD / 16; ++mt) w.run.out[mt][h] = w.run.out[mt][2 + h] = 0.0F;
    }
    float* scores = plan.scores ? plan.scores + (static_cast<size_t>(s) * a.q_heads + head0) * capacity : nullptr;
    w.tokens(x, at, q, first, last, phase, phases, scores, capacity, heads_here, ring);

    // ---- merge of the warps of one kv head
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) w.run.sum[h] += __shfl_xor_sync(0xffffffffU, w.run.sum[h], o);
    __syncthreads();  // the rings of all warps have been read
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t row = warp * kHeads + 2U * w.c + h;
      if (w.r == 0U) {
        merge_max[row] = w.run.reference[h];
        merge_sum[row] = w.run.sum[h];
      }
#pragma unroll
      for (int mt = 0; mt < HD / 16; ++mt)
        *reinterpret_cast<float2*>(merge_out + row * X::kRow + L::out_dim(mt, w.r, turn)) = make_float2(w.run.out[mt][h], w.run.out[mt][2 + h]);
    }
    __syncthreads();
    const bool begins = from == 0U, whole = begins && last == length;
    if (begins && threadIdx.x == 0U) {
      const unsigned long long last_unit = u - local + n - 1ULL;
      plan.spans[static_cast<size_t>(s) * plan.items + item] =
          make_uint2(blockIdx.x, static_cast<uint32_t>(((last_unit + 1ULL) * blocks - 1ULL) / total));
    }
    float* place = plan.partials + (static_cast<size_t>(blockIdx.x) * 2U + (begins ? 1U : 0U)) * plan.place;
    // A thread takes four dimensions of one head, all loads before the first use (one dimension and one warp after the other:
    // 11.7 us instead of 9.8 us for 1 x 1000, 144 us instead of 136 us for 96 ragged sequences).
    for (uint32_t h = 0; h < plan.heads; ++h)
      for (uint32_t e = threadIdx.x; e < heads_here * (HD / 4U); e += kThreads) {
        const uint32_t d = 4U * (e % (HD / 4U)), g = e / (HD / 4U);
        float tops[kWarps], sums[kWarps], top = -INFINITY;
        float4 outs[kWarps];
#pragma unroll
        for (uint32_t p = 0; p < kWarps; ++p) {
          const uint32_t row = (p * plan.heads + h) * kHeads + g;
          const bool there = p < phases;
          tops[p] = there ? merge_max[row] : -INFINITY;
          sums[p] = there ? merge_sum[row] : 0.0F;
          outs[p] = there ? *reinterpret_cast<const float4*>(merge_out + row * X::kRow + d) : make_float4(0.0F, 0.0F, 0.0F, 0.0F);
          top = fmaxf(top, tops[p]);
        }
        const float reference = top == -INFINITY ? 0.0F : top;
        float sum = 0.0F;
        float4 out = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
#pragma unroll
        for (uint32_t p = 0; p < kWarps; ++p) {
          const float f = exp2_fast(tops[p] - reference);
          sum = fmaf(sums[p], f, sum);  // 0 where no key counts, NaN where a score was NaN
          add_scaled(out, outs[p], f);
        }
        const uint32_t head = (set * plan.heads + h) * plan.group + tile * kHeads + g;
        if (whole) {
          put_four(static_cast<T*>(a.out) + static_cast<size_t>(s) * a.out_stride + static_cast<size_t>(head) * HD + d, out, sum);
          if (plan.lse && d == 0U) plan.lse[static_cast<size_t>(s) * a.q_heads + head] = sum == 0.0F ? 0.0F : reference + log2f(sum);
        } else {
          const uint32_t row = h * kHeads + g;
          *reinterpret_cast<float4*>(place + 2U * plan.rows + row * HD + d) = out;
          if (d == 0U) {
            place[row] = top;
            place[plan.rows + row] = sum;
          }
        }
      }
    u += take;
  }
}

// Second launch.  Its last blocks join the parts of the items that lie in more than one share, and write the zeros of
// the sequences without tokens: kWays warps to a query head, four (the warps of a block; long sequences of many parts) or one (many
// sequences of few parts: a block per head costs a chain of four loads for two or three parts).  A warp takes every
// kWays-th part, a lane four dimensions of it, and every lane works out the factors of the parts it broadcasts.
// The blocks before them, `chunks` to a kv head, add up the weights: scores and log-sums are in the workspace.
__device__ __forceinline__ const float* place_of(const Plan& plan, uint2 span, uint32_t i) {
  return plan.partials + (static_cast<size_t>(span.x + i) * 2U + (i == 0U ? 1U : 0U)) * plan.place;
}
__device__ __forceinline__ uint2 span_of(const Plan& plan, uint32_t s, uint32_t kv_head, uint32_t g) {
  return plan.spans[static_cast<size_t>(s) * plan.items + kv_head / plan.heads * plan.tiles + g / kHeads];
}
// Maximum over the parts (their reference, log2) and, in the lanes, parts of the sum.
__device__ __forceinline__ float top_of(const Plan& plan, uint2 span, uint32_t row, uint32_t lane) {
  float top = -INFINITY;
  for (uint32_t i = lane; i < span.y - span.x + 1U; i += 32U) top = fmaxf(top, place_of(plan, span, i)[row]);
  return warp_max(top);
}

template <typename T, int HD, uint32_t kWays>
__device__ __forceinline__ void join_head(const DecodeAttentionArgs& a, const Plan& plan, uint32_t s, uint32_t head, uint32_t way) {
  constexpr uint32_t kVectors = (HD + 127) / 128;         // of four dimensions a lane holds
  __shared__ float4 part[kWays > 1U ? kWays : 1U][kWays > 1U ? HD / 4 : 1];
  T* out = static_cast<T*>(a.out) + static_cast<size_t>(s) * a.out_stride + static_cast<size_t>(head) * HD;
  const uint32_t lane = threadIdx.x & 31U;
  const uint32_t kv_head = head / plan.group, g = head % plan.group;
  const uint2 span = span_of(plan, s, kv_head, g);  // together with the length; of no meaning where that is zero
  if (a.lengths[s] == 0U) {
    for (uint32_t d = way * 32U + lane; d < HD; d += 32U * kWays) put_row(out + d, 0.0F);
    return;
  }
  const uint32_t count = span.y - span.x + 1U;
  if (count <= 1U) return;
  const uint32_t row = (kv_head % plan.heads) * kHeads + g % kHeads;
  // lane i has maximum and sum of parts 32 c + i: of the first 32 kChunks parts all at once, one chunk after the other behind them
  constexpr uint32_t kChunks = 3;
  float of_part[kChunks], sum_of_part[kChunks], top = -INFINITY;
#pragma unroll
  for (uint32_t c = 0; c < kChunks; ++c) {
    const bool there = 32U * c + lane < count;
    of_part[c] = there ? place_of(plan, span, 32U * c + lane)[row] : -INFINITY;
    sum_of_part[c] = there ? place_of(plan, span, 32U * c + lane)[plan.rows + row] : 0.0F;
    top = fmaxf(top, of_part[c]);
  }
  top = count <= 32U * kChunks ? warp_max(top) : top_of(plan, span, row, lane);
  const float reference = top == -INFINITY ? 0.0F : top;
  float sum = 0.0F;
  float4 acc[kVectors];
#pragma unroll
  for (uint32_t v = 0; v < kVectors; ++v) acc[v] = make_float4(0.0F, 0.0F, 0.0F, 0.0F);
  const auto add_chunk = [&](uint32_t i0, float of_lane, float sum_of_lane) {  // each warp adds its own parts
    const float factor = exp2_fast(of_lane - reference);
    sum = fmaf(sum_of_lane, factor, sum);
    const uint32_t here = min(32U, count - i0);
#pragma unroll 8
    for (uint32_t i = way; i < here; i += kWays) {
      const float f = __shfl_sync(0xffffffffU, factor, i);
      const float4* from = reinterpret_cast<const float4*>(place_of(plan, span, i0 + i) + 2U * plan.rows + row * HD);
#pragma unroll
      for (uint32_t v = 0; v < kVectors; ++v)
        if (lane + 32U * v < HD / 4) add_scaled(acc[v], from[lane + 32U * v], f);
    }
  };
#pragma unroll
  for (uint32_t c = 0; c < kChunks; ++c)
    if (32U * c < count) add_chunk(32U * c, of_part[c], sum_of_part[c]);
  for (uint32_t i0 = 32U * kChunks; i0 < count; i0 += 32U) {
    const bool there = i0 + lane < count;
    add_chunk(i0, there ? place_of(plan, span, i0 + lane)[row] : -INFINITY, there ? place_of(plan, span, i0 + lane)[plan.rows + row] : 0.0F);
  }
  sum = warp_sum(sum);
  if constexpr (kWays > 1U) {
#pragma unroll
    for (uint32_t v = 0; v < kVectors; ++v)
      if (lane + 32U * v < HD / 4) part[way][lane + 32U * v] = acc[v];
    __syncthreads();
    for (uint32_t d = way * 32U + lane; d < HD; d += 32U * kWays) {
      float total = 0.0F;
#pragma unroll
      for (uint32_t w = 0; w < kWays; ++w) total += reinterpret_cast<const float*>(part[w])[d];
      put_row(out + d, sum == 0.0F ? 0.0F : total / sum);
    }
  } else {
#pragma unroll
    for (uint32_t v = 0; v < kVectors; ++v)
      if (lane + 32U * v < HD / 4) put_four(out + 4U * (lane + 32U * v), acc[v], sum);
  }
}

__device__ __forceinline__ void add_weights(const DecodeAttentionArgs& a, const Plan& plan, uint32_t s, uint32_t h, uint32_t chunk, uint32_t chunks) {
  __shared__ float lse[kHeads];
  constexpr uint32_t kEach = kWeightTokens / kThreads;
  const uint32_t lane = threadIdx.x & 31U, warp = threadIdx.x >> 5U;
  const uint32_t capacity = kv_capacity(a.cache), n = min(a.lengths[s], capacity);
  if (chunk * kWeightTokens >= n) return;
  const size_t row = (static_cast<size_t>(s) * a.cache.kv_heads + h) * a.weights_stride;
  for (uint32_t g0 = 0; g0 < plan.group; g0 += kHeads) {
    const uint32_t here = min(kHeads, plan.group - g0);
    const uint32_t head0 = h * plan.group + g0;
    const uint2 span = span_of(plan, s, h, g0);
    __syncthreads();
    for (uint32_t g = warp; g < here; g += kThreads / 32U) {
      float value;
      if (span.x == span.y) {
        value = plan.lse[static_cast<size_t>(s) * a.q_heads + head0 + g];
      } else {
        const uint32_t place_row = (h % plan.heads) * kHeads + g;
        const float top = top_of(plan, span, place_row, lane);
        const float reference = top == -INFINITY ? 0.0F : top;
        float total = 0.0F;
        for (uint32_t i = lane; i < span.y - span.x + 1U; i += 32U)
          total += place_of(plan, span, i)[plan.rows + place_row] * exp2_fast(place_of(plan, span, i)[place_row] - reference);
        total = warp_sum(total);
        value = total == 0.0F ? 0.0F : reference + log2f(total);
      }
      if (lane == 0U) lse[g] = value;
    }
    __syncthreads();
    const float* scores = plan.scores + (static_cast<size_t>(s) * a.q_heads + head0) * capacity + threadIdx.x;
    const float* start = g0 ? a.weights_out : a.weights_in;
    for (uint32_t t0 = chunk * kWeightTokens; t0 < n; t0 += chunks * kWeightTokens) {
      const uint32_t left = n - t0;  // tokens from here on
      float added[kEach], score[kHeads][kEach];
#pragma unroll
      for (uint32_t g = 0; g < kHeads; ++g) {
        if (g >= here) break;
        const float* from = scores + static_cast<size_t>(g) * capacity + t0;
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) score[g][i] = i * kThreads + threadIdx.x < left ? from[i * kThreads] : 0.0F;
      }
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i)
        added[i] = start && i * kThreads + threadIdx.x < left ? start[row + t0 + i * kThreads + threadIdx.x] : 0.0F;
      float sum[kEach] = {};
#pragma unroll
      for (uint32_t g = 0; g < kHeads; ++g) {
        if (g >= here) break;
        const float of = lse[g];
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) sum[i] += exp2_fast(score[g][i] - of);
      }
      float* to = a.weights_out + row + t0 + threadIdx.x;
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i)
        if (i * kThreads + threadIdx.x < left) to[i * kThreads] = added[i] + sum[i];
    }
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 8) decode_join_kernel(const __grid_constant__ DecodeAttentionArgs a, const __grid_constant__ Plan plan,
                                                               uint32_t joins, uint32_t ways, uint32_t chunks) {
  pdl_wait();
  const uint32_t warp = threadIdx.x >> 5U, first_join = gridDim.x - joins;
  if (blockIdx.x < first_join) {
    const uint32_t row = blockIdx.x / chunks;
    add_weights(a, plan, row / a.cache.kv_heads, row % a.cache.kv_heads, blockIdx.x % chunks, chunks);
    return;
  }
  const uint32_t block = blockIdx.x - first_join;
  if (ways == kWarps) {
    join_head<T, HD, kWarps>(a, plan, block / a.q_heads, block % a.q_heads, warp);
  } else {
    const uint32_t head = block * kWarps + warp;
    if (head < a.cache.sequences * a.q_heads) join_head<T, HD, 1>(a, plan, head / a.q_heads, head % a.q_heads, 0U);
  }
}

int multiprocessors(uint32_t* count) {
  int device = 0, n = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
  *count = static_cast<uint32_t>(n);
  return check_cuda(e, "decode_attention device");
}

template <typename T, int ENC, int HD>
int launch(const DecodeAttentionArgs& a, const Plan& plan, cudaStream_t stream) {
  using X = Traits<T, ENC, HD>;
  uint32_t sms = 0;
  int rc = multiprocessors(&sms);
  if (rc) return rc;
  if constexpr (X::kShared > kSharedByDefault) {
    rc = check_cuda(cudaFuncSetAttribute(decode_attention_kernel<T, ENC, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(X::kShared)), "decode_attention shared memory opt-in");
    if (rc) return rc;
  }
  const uint32_t grid = min(kMaxBlocks, sms * X::kBlocksPerSm);
  count_launch(2U);
  rc = check_cuda(launch_ordered(decode_attention_kernel<T, ENC, HD>, dim3(grid), dim3(kThreads), X::kShared, stream, a, plan),
                  "decode_attention");
  if (rc) return rc;
  // The first launch does not call for the second early: blocks that wait beside it made 1 x 32768 Q4H 25.2 us instead of 23.6 us.
  // Four warps to a query head as long as they find room at once, up to eight heads to a multiprocessor (up to four: 34.3 -> 35.5 us for
  // 16 x 8192 Q4H of 40 heads and 34.6 -> 36.0 for 32 x 4096 F16 of 32; up to sixteen: 89.4 -> 90.6 for 48 x 8192 Q4H and 60.5 -> 61.7 for
  // 64 x 4096 F16, 70.0 -> 68.6 for 20 x 16384 Q8 of 64).
  const uint32_t heads = a.cache.sequences * a.q_heads;
  const uint32_t ways = heads <= 8U * sms ? kWarps : 1U;
  const uint32_t joins = ways == kWarps ? heads : (heads + kWarps - 1U) / kWarps;
  uint32_t chunks = 1U, rows = 0U;
  if (plan.scores) {  // about 16 blocks to a multiprocessor (4: 170 us, 8: 164 us, 16: 163 us for 96 ragged sequences)
    rows = a.cache.sequences * a.cache.kv_heads;
    chunks = max(1U, min((16U * sms + rows - 1U) / rows, (kv_capacity(a.cache) + kWeightTokens - 1U) / kWeightTokens));
  }
  return check_cuda(launch_pdl(decode_join_kernel<T, HD>, dim3(joins + rows * chunks), dim3(kThreads), 0, stream, a, plan, joins, ways, chunks),
                    "decode_attention join");
}

template <typename T, int ENC>
int dispatch_dim(const DecodeAttentionArgs& a, const Plan& plan, cudaStream_t stream) {
  switch (a.cache.head_dim) {
    case 64: return launch<T, ENC, 64>(a, plan, stream);
    case 128: return launch<T, ENC, 128>(a, plan, stream);
    case 192: return launch<T, ENC, 192>(a, plan, stream);
    default: return launch<T, ENC, 256>(a, plan, stream);
  }
}
template <typename T>
int dispatch(const DecodeAttentionArgs& a, const Plan& plan, cudaStream_t stream) {
  if (a.cache.encoding == QLLM_KV_F16) return dispatch_dim<T, QLLM_KV_F16>(a, plan, stream);
  if (a.cache.encoding == QLLM_KV_Q4H) return dispatch_dim<T, QLLM_KV_Q4H>(a, plan, stream);
  return dispatch_dim<T, QLLM_KV_Q8>(a, plan, stream);
}

}  // namespace

size_t decode_attention_workspace_bytes(const KvBatch& c, uint32_t q_heads, bool weights) {
  return plan_of(c, q_heads, weights, nullptr).bytes;
}

int launch_decode_attention(const DecodeAttentionArgs& a, cudaStream_t stream) {
  const Plan plan = plan_of(a.cache, a.q_heads, a.weights_out != nullptr, a.workspace);
  if (a.row_type == QLLM_ROW_F32) return dispatch<float>(a, plan, stream);
  if (a.row_type == QLLM_ROW_BF16) return dispatch<__nv_bfloat16>(a, plan, stream);
  return dispatch<__half>(a, plan, stream);
}

}  // namespace qllm
