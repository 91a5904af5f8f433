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
// Inner product on the tensor cores (mma.sync m16n8k16, F16 in, FP32 out) with the CACHE as the M operand:
// S^T = K q^T has 16 keys x 8 heads, out^T = V^T P^T 16 dims x 8 heads, so that a group of up to eight query
// heads fills the N = 8 side instead of a sixteenth to a half of an M side.  tcgen05 wants an M of 64 or 128
// and its operands in shared memory; here the keys go from global memory straight into the registers of a
// fragment (no shared memory, no barrier) because the order of k inside a product is free: a lane takes
// whichever 16 bytes of a row it can load at once, and the query is laid out to match.  For V^T the pairs
// of keys that a fragment packs are put together by byte permutes.  Key 2 r stands in row r of a 16-key
// block, key 2 r + 1 in row r + 8, so that a lane's two keys (scales, scores) are neighbours.
//
// Numerics: codes of Q8 and Q4H records are small integers, exact in F16; their scales multiply scores and
// weights in FP32.  A query row is scaled by a power of two to [2^8, 2^9) before it becomes F16, so BF16 rows
// lose nothing that FP32 sums would keep; FP32 rows become two F16 terms (22 bits), and so do the weights
// p that meet V.  With 16-bit rows p is one F16 term: 2^-11 of each weight, below the rounding of a BF16 row and
// equal to that of an F16 row before averaging.  The softmax reference is only moved when p would exceed 2^15 (one
// vote per tile instead of a reduction) and is set so that the largest p is 2^7 then: F16 holds p down to 2^-32 of
// the largest, and a quantised V's scale is counted into the reference so that this holds for p times scale.
#include "kv_batch.cuh"
#include "launch.cuh"

namespace qllm {

namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kThreads = 32 * kWarps;
constexpr uint32_t kUnit = 64;          // tokens
constexpr uint32_t kMaxBlocks = 512;    // of the first launch; places in the workspace
constexpr uint32_t kHeads = 8;          // query heads of an item per kv head
constexpr uint32_t kJoinThreads = 256;
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
  size_t place;            // floats of one place: heads * 8 * (2 + head_dim)
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
  p.place = static_cast<size_t>(p.heads) * kHeads * (2U + c.head_dim);
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
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// Four nibbles (two's complement) at bits 0, 4, 8, 12 of each 16-bit half -> pairs of F16, one per nibble position:
// 0x6400 | (n ^ 8) is 1024 + n + 8, and with the nibble four bits higher 1024 + 16 (n + 8).
__device__ __forceinline__ void nibbles_to_half(uint32_t w, uint32_t (&h)[4]) {
  const uint32_t high = w >> 8U;
  h[0] = half2_sub(mask_flip<0x000F000FU, 0x64086408U>(w), 0x64086408U);
  h[1] = half2_fma(mask_flip<0x00F000F0U, 0x64806480U>(w), 0x2C002C00U, 0xD480D480U);      // / 16 - 72
  h[2] = half2_sub(mask_flip<0x000F000FU, 0x64086408U>(high), 0x64086408U);
  h[3] = half2_fma(mask_flip<0x00F000F0U, 0x64806480U>(high), 0x2C002C00U, 0xD480D480U);
}
// Signed bytes in bits 0-7 of each half -> F16: 0x6400 | (b ^ 0x80) is 1024 + b + 128.
__device__ __forceinline__ uint32_t bytes_to_half(uint32_t v) {
  return half2_sub(mask_flip<0x00FF00FFU, 0x64806480U>(v), 0x64806480U);
}

// ---- what depends on the encoding: how a lane's registers hold a 16-key block.
// lane = 4 r + c.  K: rows r (key 2 r) and r + 8 (key 2 r + 1).  V: keys 4 c .. 4 c + 3.
template <int ENC, int HD>
struct Layout {
  static constexpr bool kStaged = ENC == QLLM_KV_Q8;
  // blocks of 16 keys that a warp takes at a time: 32 registers of K and of V (HD 64, 128, 256), 24 - 48 (192)
  static constexpr int kBlocks = ENC == QLLM_KV_F16 ? (HD == 64 ? 2 : 1) : ENC == QLLM_KV_Q4H ? (HD <= 128 ? 4 : 2) : 1;
  static constexpr int kRegs = ENC == QLLM_KV_F16 ? HD / 4 : ENC == QLLM_KV_Q4H ? HD / 16 : 1;  // of K, and of V, per block
  static constexpr int kKWords = ENC == QLLM_KV_Q4H ? (HD % 128 == 0 ? 4 : 2) : 4;      // words per load
  static constexpr int kVWords = ENC == QLLM_KV_Q4H ? (HD == 128 ? 2 : HD == 256 ? 4 : 1) : 4;
  // staged rows: the 16-byte windows that cover a record wherever it begins
  static constexpr int kWindows = HD / 16 + 1;
  static constexpr int kPitch = 16 * kWindows;
  static constexpr int kStage = 2 * 16 * kPitch;
  static constexpr int kStages = HD == 64 ? 4 : HD <= 192 ? 3 : 2;  // as many as leave room for kBlocksPerSm

  // dimensions of half-words 0 and 1 of fragment register b (0, 1) in k step `ks`, lane c
  static __device__ __forceinline__ uint32_t query_dim(int ks, int b, int half, uint32_t c) {
    if constexpr (ENC == QLLM_KV_F16) return 8U * (c + 4U * (ks / 2)) + 4U * (ks % 2) + 2U * b + half;
    if constexpr (ENC == QLLM_KV_Q8) return 2U * (c + 4U * (2 * ks + b)) + half;
    const uint32_t word = (c + 4U * (ks / 2 / kKWords)) * kKWords + (ks / 2) % kKWords;
    return 8U * word + 2U * (ks % 2) + b + 4U * half;
  }
  // first of the two neighbouring dimensions of output tile mt in lane r
  static __device__ __forceinline__ uint32_t out_dim(int mt, uint32_t r) {
    if constexpr (ENC == QLLM_KV_F16) return 8U * (r + 8U * (mt / 4)) + 2U * (mt % 4);
    if constexpr (ENC == QLLM_KV_Q8) return 2U * (r + 8U * mt);
    const uint32_t word = (r + 8U * (mt / 4 / kVWords)) * kVWords + (mt / 4) % kVWords;
    return 8U * word + 2U * (mt % 4);
  }
};

// Where the keys of a 16-key block lie.
struct Block {
  const uint8_t* layer;  // null: no page
  uint32_t place;        // of its first token in the page
  uint32_t count;        // keys that count, 0..16
};

template <typename T, int ENC, int HD>
struct Traits {
  static constexpr bool kPrecise = sizeof(T) == 4;
  static constexpr int kTerms = kPrecise ? 2 : 1;
  static constexpr int kSteps = HD / 16;
  static constexpr bool kQueryInRegisters = HD <= 128;
  static constexpr int kBlocksPerSm = HD <= 128 ? 3 : 2;
  static constexpr size_t kFragmentBytes = static_cast<size_t>(kSteps) * 32 * kTerms * sizeof(uint2);  // of one kv head
  static constexpr int kRow = HD + 4;  // floats of one head in the merge area
  static constexpr size_t kMergeBytes = (kWarps * kHeads * kRow + 2 * kWarps * kHeads) * sizeof(float);
  static constexpr size_t kRingBytes = Layout<ENC, HD>::kStaged ? static_cast<size_t>(kWarps) * Layout<ENC, HD>::kStages * Layout<ENC, HD>::kStage : 0;
  static constexpr size_t kShared = (kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes) + kFragmentBytes * (ENC == QLLM_KV_Q8 ? 4 : 1);
};

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
    for (int k = 0; k < 2; ++k) bias[b][k] = kScaled ? __log2f(fmaxf(fabsf(vscale[b][k]), 0x1p-24F)) : 0.0F;
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

// Weights of a block as the B operand (keys x heads), one or two F16 terms.
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

__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from, bool there) {
  const uint32_t bytes = there ? 16U : 0U;  // 0: the 16 bytes become zero and nothing is read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// Block `index` of the warp's blocks in tokens [first, last) of a sequence.
__device__ __forceinline__ Block find_block(const KvBatch& c, uint32_t sequence, uint32_t first, uint32_t last, uint32_t index,
                                            uint32_t phase, uint32_t phases) {
  const uint64_t t = first + 16ULL * (phase + static_cast<uint64_t>(phases) * index);
  Block b{nullptr, 0U, 0U};
  if (t < last) {
    const uint32_t page = static_cast<uint32_t>(t) / c.page_tokens;
    b.place = static_cast<uint32_t>(t) - page * c.page_tokens;
    b.layer = kv_page(c, sequence, page);
    b.count = b.layer ? min(16U, last - static_cast<uint32_t>(t)) : 0U;
  }
  return b;
}
__device__ __forceinline__ Block take_block(const Block& mine, int lane) {
  Block b;
  b.layer = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffU, reinterpret_cast<unsigned long long>(mine.layer), lane));
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

  // ---- registers (F16, Q4H)
  __device__ __forceinline__ void load_keys(const Block& b, uint32_t (&k)[L::kRegs], uint32_t& scales) {
    if (b.count == 0U) {
#pragma unroll
      for (int i = 0; i < L::kRegs; ++i) k[i] = 0U;
      scales = 0U;
      return;
    }
    if constexpr (ENC == QLLM_KV_F16) {
      const size_t stride = static_cast<size_t>(a.cache.kv_heads) * HD * 2U;
      const uint8_t* p = b.layer + (b.place + 2U * r) * stride + static_cast<size_t>(kv_head) * HD * 2U + 16U * c;
#pragma unroll
      for (int row = 0; row < 2; ++row)
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) load_words<4>(&k[row * (HD / 8) + 4 * j], p + row * stride + 64 * j);
    } else {
      const size_t record = static_cast<size_t>(kv_head) * a.cache.page_tokens + b.place + 2U * r;
      const uint8_t* p = b.layer + record * (HD / 2) + 4 * L::kKWords * c;
#pragma unroll
      for (int row = 0; row < 2; ++row)
#pragma unroll
        for (int j = 0; j < HD / 32 / L::kKWords; ++j)
          load_words<L::kKWords>(&k[row * (HD / 32) + L::kKWords * j], p + row * (HD / 2) + 16 * L::kKWords * j);
      load_words<1>(&scales, b.layer + static_cast<size_t>(a.cache.page_tokens) * a.cache.kv_heads * (HD / 2) + record * 2U);
    }
  }
  __device__ __forceinline__ void load_values(const Block& b, uint32_t (&v)[L::kRegs], uint32_t& scales) {
    const size_t records = static_cast<size_t>(a.cache.page_tokens) * a.cache.kv_heads;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool there = 4U * c + q < b.count;
      if constexpr (ENC == QLLM_KV_F16) {
        const size_t stride = static_cast<size_t>(a.cache.kv_heads) * HD * 2U;
        const uint8_t* p = b.layer + records * HD * 2U + (b.place + 4U * c + q) * stride + static_cast<size_t>(kv_head) * HD * 2U + 16U * r;
#pragma unroll
        for (int j = 0; j < HD / 64; ++j) {
          uint32_t* d = &v[(q * (HD / 64) + j) * 4];
          d[0] = d[1] = d[2] = d[3] = 0U;
          if (there) load_words<4>(d, p + 128 * j);
        }
      } else {
        const size_t record = static_cast<size_t>(kv_head) * a.cache.page_tokens + b.place + 4U * c + q;
        const uint8_t* p = b.layer + records * (HD / 2 + 2) + record * (HD / 2) + 4 * L::kVWords * r;
#pragma unroll
        for (int j = 0; j < HD / 64 / L::kVWords; ++j) {
          uint32_t* d = &v[q * (HD / 64) + L::kVWords * j];
#pragma unroll
          for (int i = 0; i < L::kVWords; ++i) d[i] = 0U;
          if (there) load_words<L::kVWords>(d, p + 32 * L::kVWords * j);
        }
      }
    }
    scales = 0U;
    if constexpr (ENC == QLLM_KV_Q4H) {
      if (b.count) {
        const size_t record = static_cast<size_t>(kv_head) * a.cache.page_tokens + b.place + 2U * r;
        load_words<1>(&scales, b.layer + records * (HD / 2 + 2) + records * (HD / 2) + record * 2U);
      }
    }
  }
  template <int kQ>
  __device__ __forceinline__ void score(const uint2 (&q)[kQ], const uint32_t (&k)[L::kRegs], float (&s)[4]) const {
    s[0] = s[1] = s[2] = s[3] = 0.0F;
#pragma unroll
    for (int w = 0; w < X::kSteps / 2; ++w) {
      uint32_t lo[4], hi[4];
      if constexpr (ENC == QLLM_KV_F16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = k[4 * w + i];
          hi[i] = k[HD / 8 + 4 * w + i];
        }
      } else {
        nibbles_to_half(k[w], lo);
        nibbles_to_half(k[HD / 32 + w], hi);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int term = 0; term < X::kTerms; ++term) {
          const uint2 f = query(q, 2 * w + half, term);
          mma16816(s, lo[2 * half], hi[2 * half], lo[2 * half + 1], hi[2 * half + 1], f.x, f.y);
        }
    }
  }
  __device__ __forceinline__ void add_values(const uint32_t (&v)[L::kRegs], const float (&p)[4]) {
    uint32_t hi[2], lo[2] = {0U, 0U};
    weight_fragments<X::kPrecise>(p, hi, lo);
    // keys 4c, 4c+2 are k = 2c, 2c+1 of the product, keys 4c+1, 4c+3 k = 2c+8, 2c+9
#pragma unroll
    for (int w = 0; w < HD / 64; ++w) {
      if constexpr (ENC == QLLM_KV_F16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t k0 = v[w * 4 + i], k1 = v[(HD / 64 + w) * 4 + i];
          const uint32_t k2 = v[(2 * (HD / 64) + w) * 4 + i], k3 = v[(3 * (HD / 64) + w) * 4 + i];
          const uint32_t a0 = __byte_perm(k0, k2, 0x5410), a1 = __byte_perm(k0, k2, 0x7632);
          const uint32_t a2 = __byte_perm(k1, k3, 0x5410), a3 = __byte_perm(k1, k3, 0x7632);
          mma16816(run.out[4 * w + i], a0, a1, a2, a3, hi[0], hi[1]);
          if constexpr (X::kPrecise) mma16816(run.out[4 * w + i], a0, a1, a2, a3, lo[0], lo[1]);
        }
      } else {
        const uint32_t k0 = v[w], k1 = v[HD / 64 + w], k2 = v[2 * (HD / 64) + w], k3 = v[3 * (HD / 64) + w];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t selector = half ? 0x7632U : 0x5410U;
          uint32_t even[4], odd[4];
          nibbles_to_half(__byte_perm(k0, k2, selector), even);
          nibbles_to_half(__byte_perm(k1, k3, selector), odd);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int mt = 4 * w + 2 * half + i;
            mma16816(run.out[mt], even[2 * i], even[2 * i + 1], odd[2 * i], odd[2 * i + 1], hi[0], hi[1]);
            if constexpr (X::kPrecise) mma16816(run.out[mt], even[2 * i], even[2 * i + 1], odd[2 * i], odd[2 * i + 1], lo[0], lo[1]);
          }
        }
      }
    }
  }

  // ---- through shared memory (Q8): rows of windows, key 2r in row r, key 2r + 1 in row r + 8
  __device__ __forceinline__ void stage(const Block& b, uint32_t to) {
    const size_t stride = static_cast<size_t>(a.cache.kv_heads) * (HD + 2);
    const size_t records = static_cast<size_t>(a.cache.page_tokens) * a.cache.kv_heads;
    const uint8_t* base = b.layer + b.place * stride + static_cast<size_t>(kv_head) * (HD + 2);
#pragma unroll
    for (int value = 0; value < 2; ++value)
      for (uint32_t i = lane; i < 16U * L::kWindows; i += 32U) {
        const uint32_t key = i / L::kWindows, window = i % L::kWindows;
        const uintptr_t record = reinterpret_cast<uintptr_t>(base + value * records * (HD + 2) + key * stride);
        const uint32_t row = value * 16U + key / 2U + 8U * (key & 1U);
        const bool there = key < b.count;
        copy16(to + row * L::kPitch + 16U * window,
               there ? reinterpret_cast<const uint8_t*>(record & ~static_cast<uintptr_t>(15U)) + 16U * window
                     : reinterpret_cast<const uint8_t*>(a.cache.page_tables), there);
      }
  }
  // where a record begins in its row
  __device__ __forceinline__ uint32_t shift_of(const Block& b, uint32_t key, bool value) const {
    const size_t stride = static_cast<size_t>(a.cache.kv_heads) * (HD + 2);
    const size_t records = static_cast<size_t>(a.cache.page_tokens) * a.cache.kv_heads;
    return static_cast<uint32_t>((b.place + key) * stride + static_cast<size_t>(kv_head) * (HD + 2) +
                                 (value ? records * (HD + 2) : 0U)) & 15U;  // pages and layers begin on 16 bytes
  }

  // Tokens [first, last) of the sequence, every `phases`-th block of 16 from `phase` on.
  template <int kQ>
  __device__ __forceinline__ void tokens(const uint2 (&q)[kQ], uint32_t first, uint32_t last, uint32_t phase, uint32_t phases,
                                         float* scores, size_t capacity, uint32_t heads_here, uint8_t* ring) {
    const uint32_t blocks = (last - first + 15U) / 16U;
    const uint32_t mine = blocks > phase ? (blocks - phase + phases - 1U) / phases : 0U;
    const uint32_t tiles = (mine + kN - 1U) / kN;
    if constexpr (!L::kStaged) {
      uint32_t k[kN][L::kRegs], v[kN][L::kRegs], kscale[kN], vscale[kN];
      Block now[kN];
      Block ahead = find_block(a.cache, sequence, first, last, lane % kN, phase, phases);
#pragma unroll
      for (int b = 0; b < kN; ++b) {
        now[b] = take_block(ahead, b);
        load_keys(now[b], k[b], kscale[b]);
      }
#pragma unroll
      for (int b = 0; b < kN; ++b) load_values(now[b], v[b], vscale[b]);
      ahead = find_block(a.cache, sequence, first, last, kN + lane % kN, phase, phases);
      for (uint32_t tile = 0; tile < tiles; ++tile) {
        float s[kN][4], vs[kN][2];
        uint32_t count[kN];
#pragma unroll
        for (int b = 0; b < kN; ++b) {
          score(q, k[b], s[b]);
          count[b] = now[b].count;
          const float2 ks = ENC == QLLM_KV_Q4H ? unpack_half(kscale[b]) : make_float2(1.0F, 1.0F);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            s[b][h] = 2U * r < count[b] ? s[b][h] * (ks.x * scale[h]) : -INFINITY;
            s[b][2 + h] = 2U * r + 1U < count[b] ? s[b][2 + h] * (ks.y * scale[h]) : -INFINITY;
          }
          put_scores(scores, capacity, heads_here, first + 16U * (phase + phases * (tile * kN + b)), last, s[b]);
        }
        const bool more = tile + 1U < tiles;
        if (more) {
#pragma unroll
          for (int b = 0; b < kN; ++b) {
            now[b] = take_block(ahead, b);
            load_keys(now[b], k[b], kscale[b]);
          }
        }
#pragma unroll
        for (int b = 0; b < kN; ++b) {
          const float2 f = ENC == QLLM_KV_Q4H ? unpack_half(vscale[b]) : make_float2(1.0F, 1.0F);
          vs[b][0] = 2U * r < count[b] ? f.x : 0.0F;
          vs[b][1] = 2U * r + 1U < count[b] ? f.y : 0.0F;
        }
        softmax_tile<HD, kN, ENC != QLLM_KV_F16>(run, s, vs);
#pragma unroll
        for (int b = 0; b < kN; ++b) add_values(v[b], s[b]);
        if (more) {
#pragma unroll
          for (int b = 0; b < kN; ++b) load_values(now[b], v[b], vscale[b]);
          ahead = find_block(a.cache, sequence, first, last, (tile + 2U) * kN + lane % kN, phase, phases);
        }
      }
    } else {
      const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
      Block held[L::kStages];
#pragma unroll
      for (int i = 0; i < L::kStages - 1; ++i) {
        held[i] = find_block(a.cache, sequence, first, last, i, phase, phases);
        if (static_cast<uint32_t>(i) < tiles) stage(held[i], base + i * L::kStage);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      Block ahead = find_block(a.cache, sequence, first, last, L::kStages - 1, phase, phases);
      for (uint32_t tile0 = 0; tile0 < tiles; tile0 += L::kStages) {
#pragma unroll
        for (int i = 0; i < L::kStages; ++i) {
          const uint32_t tile = tile0 + i;
          if (tile >= tiles) break;
          asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 2) : "memory");
          __syncwarp();
          staged_block(q, held[i], ring + i * L::kStage, first + 16U * (phase + phases * tile), last, scores, capacity, heads_here);
          __syncwarp();
          constexpr int kBehind = L::kStages - 1;
          held[(i + kBehind) % L::kStages] = ahead;
          if (tile + kBehind < tiles) stage(ahead, base + (i + kBehind) % L::kStages * L::kStage);
          asm volatile("cp.async.commit_group;" ::: "memory");
          ahead = find_block(a.cache, sequence, first, last, tile + kBehind + 1U, phase, phases);
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  }
  __device__ __forceinline__ void put_scores(float* scores, size_t capacity, uint32_t heads_here, uint64_t token, uint32_t last,
                                             const float (&s)[4]) const {
    if (!scores) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (2U * c + h >= heads_here) continue;
      float* to = scores + (2U * c + h) * capacity + token + 2U * r;
      if (token + 2U * r < last) to[0] = s[h];
      if (token + 2U * r + 1U < last) to[1] = s[2 + h];
    }
  }
  template <int kQ>
  __device__ __forceinline__ void staged_block(const uint2 (&q)[kQ], const Block& b, const uint8_t* at, uint32_t token, uint32_t last,
                                               float* scores, size_t capacity, uint32_t heads_here) {
    float s[1][4] = {{0.0F, 0.0F, 0.0F, 0.0F}}, vs[1][2], ks[2];
    const uint8_t* rows[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      rows[k] = at + (r + 8U * k) * L::kPitch + shift_of(b, 2U * r + k, false);
      ks[k] = __half2float(*reinterpret_cast<const __half*>(rows[k] + HD));
      const uint8_t* value = at + (16U + r + 8U * k) * L::kPitch + shift_of(b, 2U * r + k, true);
      vs[0][k] = 2U * r + k < b.count ? __half2float(*reinterpret_cast<const __half*>(value + HD)) : 0.0F;
    }
#pragma unroll
    for (int step = 0; step < X::kSteps; ++step) {
      uint32_t x[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t pair = *reinterpret_cast<const uint16_t*>(rows[k] + 2U * (c + 4U * (2 * step + half)));
          x[k][half] = bytes_to_half(__byte_perm(pair, 0U, 0x4140));
        }
#pragma unroll
      for (int term = 0; term < X::kTerms; ++term) {
        const uint2 f = query(q, step, term);
        mma16816(s[0], x[0][0], x[1][0], x[0][1], x[1][1], f.x, f.y);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) s[0][2 * k + h] = 2U * r + k < b.count ? s[0][2 * k + h] * (ks[k] * scale[h]) : -INFINITY;
    put_scores(scores, capacity, heads_here, token, last, s[0]);
    softmax_tile<HD, 1, true>(run, s, vs);
    uint32_t hi[2], lo[2] = {0U, 0U};
    weight_fragments<X::kPrecise>(s[0], hi, lo);
    const uint8_t* v[4];
#pragma unroll
    for (uint32_t k = 0; k < 4U; ++k)
      v[k] = at + (16U + 2U * c + k / 2U + 8U * (k & 1U)) * L::kPitch + shift_of(b, 4U * c + k, true) + 2U * r;
#pragma unroll
    for (int mt = 0; mt < HD / 16; ++mt) {
      uint32_t x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const uint16_t*>(v[k] + 16 * mt);
      const uint32_t even = __byte_perm(x[0], x[2], 0x5410), odd = __byte_perm(x[1], x[3], 0x5410);
      const uint32_t a0 = bytes_to_half(even), a1 = bytes_to_half(even >> 8U), a2 = bytes_to_half(odd), a3 = bytes_to_half(odd >> 8U);
      mma16816(run.out[mt], a0, a1, a2, a3, hi[0], hi[1]);
      if constexpr (X::kPrecise) mma16816(run.out[mt], a0, a1, a2, a3, lo[0], lo[1]);
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
  __shared__ float query_scale[4][kHeads];
  const uint32_t lane = threadIdx.x & 31U, warp = threadIdx.x >> 5U;
  const uint32_t capacity = kv_capacity(a.cache), sequences = a.cache.sequences;
  const auto units_of = [&](uint32_t s) { return (min(a.lengths[s], capacity) + kUnit - 1U) / kUnit; };

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
  const unsigned long long blocks = min(static_cast<unsigned long long>(gridDim.x), total);
  if (blockIdx.x >= blocks) return;
  unsigned long long u = blockIdx.x * total / blocks;
  const unsigned long long end = (blockIdx.x + 1ULL) * total / blocks;
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

  Warp<T, ENC, HD> w{a};
  w.lane = lane;
  w.r = lane >> 2U;
  w.c = lane & 3U;
  const uint32_t in_set = warp % plan.heads, phase = warp / plan.heads, phases = kWarps / plan.heads;
  uint2* fragments = reinterpret_cast<uint2*>(shared);
  uint8_t* area = shared + X::kFragmentBytes * plan.heads;
  float* merge_max = reinterpret_cast<float*>(area);           // [warp][head]
  float* merge_sum = merge_max + kWarps * kHeads;
  float* merge_out = merge_sum + kWarps * kHeads;              // [warp][head][HD + 4]
  w.fragments = fragments + in_set * (X::kFragmentBytes / sizeof(uint2));

  while (u < end) {
    const uint32_t length = min(a.lengths[s], capacity);
    const uint32_t n = (length + kUnit - 1U) / kUnit;
    if (u >= base + static_cast<unsigned long long>(n) * plan.items) {
      base += static_cast<unsigned long long>(n) * plan.items;
      ++s;
      continue;
    }
    const uint32_t item = static_cast<uint32_t>((u - base) / n), local = static_cast<uint32_t>((u - base) % n);
    const uint32_t take = static_cast<uint32_t>(min(static_cast<unsigned long long>(n - local), end - u));
    const uint32_t first = local * kUnit, last = min(length, (local + take) * kUnit);
    const uint32_t set = item / plan.tiles, tile = item % plan.tiles;
    const uint32_t heads_here = min(kHeads, plan.group - tile * kHeads);
    const uint32_t kv_head = set * plan.heads + in_set;
    const uint32_t head0 = kv_head * plan.group + tile * kHeads;  // first query head of this warp

    // ---- the query heads as fragments (one warp per kv head), scaled to [2^8, 2^9)
    __syncthreads();  // the merge area and the fragments of the item before have been read
    if (warp < plan.heads) {
      const T* q = static_cast<const T*>(a.query) + static_cast<size_t>(s) * a.query_stride + static_cast<size_t>(head0 + w.r) * HD;
      const bool there = w.r < heads_here;
      float top = 0.0F;
      for (uint32_t d = w.c; d < HD; d += 4U) top = fmaxf(top, there ? fabsf(row_value(q[d])) : 0.0F);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffU, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffU, top, 2));
      int up = 0;
      if (top > 0.0F && top < INFINITY) up = 8 - ilogbf(top);
      if (w.c == 0U) query_scale[warp][w.r] = ldexpf(a.scale * kLog2e, -up);
      uint2* to = fragments + warp * (X::kFragmentBytes / sizeof(uint2));
#pragma unroll 2
      for (int step = 0; step < X::kSteps; ++step) {
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          float x[2];
#pragma unroll
          for (int half = 0; half < 2; ++half)
            x[half] = there ? ldexpf(row_value(q[L::query_dim(step, b, half, w.c)]), up) : 0.0F;
          hi[b] = pack_half(x[0], x[1]);
          const float2 f = unpack_half(hi[b]);
          lo[b] = pack_half(x[0] - f.x, x[1] - f.y);
        }
        to[step * X::kTerms * 32 + lane] = make_uint2(hi[0], hi[1]);
        if constexpr (X::kPrecise) to[(step * X::kTerms + 1) * 32 + lane] = make_uint2(lo[0], lo[1]);
      }
    }
    __syncthreads();
    uint2 q[X::kQueryInRegisters ? X::kSteps * X::kTerms : 1];
    if constexpr (X::kQueryInRegisters) {
#pragma unroll
      for (int i = 0; i < X::kSteps * X::kTerms; ++i) q[i] = w.fragments[i * 32 + lane];
    }
    w.scale[0] = query_scale[in_set][2U * w.c];
    w.scale[1] = query_scale[in_set][2U * w.c + 1U];
    w.sequence = s;
    w.kv_head = kv_head;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w.run.reference[h] = -INFINITY;
      w.run.sum[h] = 0.0F;
#pragma unroll
      for (int mt = 0; mt < HD / 16; ++mt) w.run.out[mt][h] = w.run.out[mt][2 + h] = 0.0F;
    }
    float* scores = plan.scores ? plan.scores + (static_cast<size_t>(s) * a.q_heads + head0) * capacity : nullptr;
    w.tokens(q, first, last, phase, phases, scores, capacity, heads_here, area + warp * (L::kStages * L::kStage));

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
        *reinterpret_cast<float2*>(merge_out + row * X::kRow + L::out_dim(mt, w.r)) = make_float2(w.run.out[mt][h], w.run.out[mt][2 + h]);
    }
    __syncthreads();
    const bool begins = local == 0U, whole = begins && take == n;
    if (begins && threadIdx.x == 0U) {
      const unsigned long long last_unit = u + n - 1ULL;
      plan.spans[static_cast<size_t>(s) * plan.items + item] =
          make_uint2(blockIdx.x, static_cast<uint32_t>(((last_unit + 1ULL) * blocks - 1ULL) / total));
    }
    float* place = plan.partials + (static_cast<size_t>(blockIdx.x) * 2U + (begins ? 1U : 0U)) * plan.place;
    for (uint32_t e = threadIdx.x; e < plan.heads * heads_here * HD; e += kThreads) {
      const uint32_t d = e % HD, g = e / HD % heads_here, h = e / HD / heads_here;
      float top = -INFINITY;
      for (uint32_t p = 0; p < phases; ++p) top = fmaxf(top, merge_max[(p * plan.heads + h) * kHeads + g]);
      float sum = 0.0F, out = 0.0F;
      if (top != -INFINITY)
        for (uint32_t p = 0; p < phases; ++p) {
          const uint32_t row = (p * plan.heads + h) * kHeads + g;
          const float f = exp2_fast(merge_max[row] - top);
          sum = fmaf(merge_sum[row], f, sum);
          out = fmaf(merge_out[row * X::kRow + d], f, out);
        }
      const uint32_t head = (set * plan.heads + h) * plan.group + tile * kHeads + g;
      if (whole) {
        put_row(static_cast<T*>(a.out) + static_cast<size_t>(s) * a.out_stride + static_cast<size_t>(head) * HD + d,
                top == -INFINITY ? 0.0F : out / sum);
        if (plan.lse && d == 0U) plan.lse[static_cast<size_t>(s) * a.q_heads + head] = top == -INFINITY ? 0.0F : top + log2f(sum);
      } else {
        float* to = place + static_cast<size_t>(h * kHeads + g) * (2U + HD);
        to[2U + d] = out;
        if (d == 0U) {
          to[0] = top;
          to[1] = sum;
        }
      }
    }
    u += take;
  }
}

// One block per (sequence, query head): joins the parts of an item that lies in more than one share, and
// writes the zeros of a sequence without tokens.
template <typename T, int HD>
__global__ void __launch_bounds__(kJoinThreads) decode_join_kernel(const __grid_constant__ DecodeAttentionArgs a, const __grid_constant__ Plan plan) {
  __shared__ float factor[kMaxBlocks], reduce[kJoinThreads / 32U], part[kJoinThreads];
  pdl_wait();
  const uint32_t head = blockIdx.x % a.q_heads, s = blockIdx.x / a.q_heads;
  T* out = static_cast<T*>(a.out) + static_cast<size_t>(s) * a.out_stride + static_cast<size_t>(head) * HD;
  const uint32_t tid = threadIdx.x, lane = tid & 31U, warp = tid >> 5U;
  if (a.lengths[s] == 0U) {
    if (tid < HD) put_row(out + tid, 0.0F);
    return;
  }
  const uint32_t kv_head = head / plan.group, g = head % plan.group;
  const uint2 span = plan.spans[static_cast<size_t>(s) * plan.items + kv_head / plan.heads * plan.tiles + g / kHeads];
  const uint32_t count = span.y - span.x + 1U;
  if (count <= 1U) return;
  const float* parts = plan.partials + static_cast<size_t>((kv_head % plan.heads) * kHeads + g % kHeads) * (2U + HD);
  const auto part_of = [&](uint32_t i) { return parts + (static_cast<size_t>(span.x + i) * 2U + (i == 0U ? 1U : 0U)) * plan.place; };
  float top = -INFINITY;
  for (uint32_t i = tid; i < count; i += kJoinThreads) top = fmaxf(top, part_of(i)[0]);
  top = warp_max(top);
  if (lane == 0U) reduce[warp] = top;
  __syncthreads();
  top = reduce[0];
#pragma unroll
  for (uint32_t w = 1; w < kJoinThreads / 32U; ++w) top = fmaxf(top, reduce[w]);
  float sum = 0.0F;
  for (uint32_t i = tid; i < count; i += kJoinThreads) {
    const float f = top == -INFINITY ? 0.0F : exp2_fast(part_of(i)[0] - top);
    factor[i] = f;
    sum += part_of(i)[1] * f;
  }
  sum = warp_sum(sum);
  __syncthreads();
  if (lane == 0U) reduce[warp] = sum;
  __syncthreads();
  sum = 0.0F;
#pragma unroll
  for (uint32_t w = 0; w < kJoinThreads / 32U; ++w) sum += reduce[w];
  constexpr uint32_t kWays = kJoinThreads / HD;  // 4, 2, 1, 1
  const uint32_t d = tid % HD, way = tid / HD;
  float acc = 0.0F;
  if (way < kWays)
#pragma unroll 4
    for (uint32_t i = way; i < count; i += kWays) acc = fmaf(part_of(i)[2U + d], factor[i], acc);
  part[tid] = acc;
  __syncthreads();
  if (tid < HD) {
#pragma unroll
    for (uint32_t w = 1; w < kWays; ++w) acc += part[w * HD + tid];
    put_row(out + tid, top == -INFINITY ? 0.0F : acc / sum);
  }
  if (plan.lse && tid == 0U) plan.lse[static_cast<size_t>(s) * a.q_heads + head] = top == -INFINITY ? 0.0F : top + log2f(sum);
}

// grid (sequences * kv heads, chunks of slots)
__global__ void __launch_bounds__(kThreads) decode_weights_kernel(const __grid_constant__ DecodeAttentionArgs a, const __grid_constant__ Plan plan) {
  pdl_wait();
  const uint32_t s = blockIdx.x / a.cache.kv_heads, h = blockIdx.x % a.cache.kv_heads;
  const uint32_t capacity = kv_capacity(a.cache), n = min(a.lengths[s], capacity);
  const float* lse = plan.lse + static_cast<size_t>(s) * a.q_heads + h * plan.group;
  const float* scores = plan.scores + (static_cast<size_t>(s) * a.q_heads + h * plan.group) * capacity;
  const size_t row = static_cast<size_t>(blockIdx.x) * a.weights_stride;
  for (uint32_t t = blockIdx.y * kThreads + threadIdx.x; t < n; t += gridDim.y * kThreads) {
    float sum = 0.0F;
    for (uint32_t g = 0; g < plan.group; ++g) sum += exp2_fast(scores[g * static_cast<size_t>(capacity) + t] - lse[g]);
    a.weights_out[row + t] = (a.weights_in ? a.weights_in[row + t] : 0.0F) + sum;
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
  rc = check_cuda(cudaFuncSetAttribute(decode_attention_kernel<T, ENC, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(X::kShared)), "decode_attention shared memory opt-in");
  if (rc) return rc;
  const uint32_t grid = min(kMaxBlocks, sms * X::kBlocksPerSm);
  count_launch(plan.scores ? 3U : 2U);
  rc = check_cuda(launch_ordered(decode_attention_kernel<T, ENC, HD>, dim3(grid), dim3(kThreads), X::kShared, stream, a, plan),
                  "decode_attention");
  if (rc) return rc;
  rc = check_cuda(launch_pdl(decode_join_kernel<T, HD>, dim3(a.cache.sequences * a.q_heads), dim3(kJoinThreads), 0, stream, a, plan),
                  "decode_attention join");
  if (rc || !plan.scores) return rc;
  const uint32_t rows = a.cache.sequences * a.cache.kv_heads;
  const uint32_t chunks = min(256U, (kv_capacity(a.cache) + kThreads - 1U) / kThreads);
  return check_cuda(launch_pdl(decode_weights_kernel, dim3(rows, chunks), dim3(kThreads), 0, stream, a, plan), "decode_attention weights");
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
  if (!c.kv_heads) return 0U;
  return plan_of(c, q_heads, weights, nullptr).bytes;
}

int launch_decode_attention(const DecodeAttentionArgs& a, cudaStream_t stream) {
  const Plan plan = plan_of(a.cache, a.q_heads, a.weights_out != nullptr, a.workspace);
  if (a.row_type == QLLM_ROW_F32) return dispatch<float>(a, plan, stream);
  if (a.row_type == QLLM_ROW_BF16) return dispatch<__nv_bfloat16>(a, plan, stream);
  return dispatch<__half>(a, plan, stream);
}

}  // namespace qllm
