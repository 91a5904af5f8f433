// Eviction from the paged cache by accumulated attention weight (qllm_k_kv_evict).
//
// Per (sequence, kv head) of n slots, m = min(n, budget) are kept: first the protected ones (position
// among the last `recent` or the first `sinks`), then by weight, ties to the lower slot.  Kept slots
// below m stay where they are; the i-th freed slot below m takes the i-th kept slot at or above m.
// Sources and targets are disjoint, so the move is in place without an order between its copies,
// and no more than min(m, n - m) records move.
//
// First launch: selection, one CTA per (sequence, kv head).  The order is that of a 32-bit key, and
// the m-th largest key is found digit by digit (four histograms of eight bits); the slots are then
// walked in order once.  Second launch: the moves.
#include "kv_batch.cuh"
#include "launch.cuh"

namespace qllm {

namespace {

constexpr uint32_t kSelectThreads = 1024;
constexpr uint32_t kMoveThreads = 256;

// Workspace: [rows] headers, then [rows][most] pairs {freed slot, kept slot}.
struct RowHeader {
  uint32_t slots, kept, moves, reserved;
};
__host__ __device__ __forceinline__ uint32_t most_moves(const KvBatch& c, uint32_t budget) {
  const uint32_t capacity = kv_capacity(c);
  return capacity <= budget ? 0U : min(budget, capacity - budget);
}

__device__ __forceinline__ bool is_protected(const KvEvictArgs& a, uint32_t position, uint32_t next) {
  return static_cast<uint64_t>(position) + a.recent >= next || position < a.sinks;
}
// Larger key = kept first: protected slots, then by weight (NaN counts as -infinity, -0 as +0).  `crowded`: more slots
// are protected than can be kept (positions that occur more than once), so the weight decides among those alone.
__device__ __forceinline__ uint32_t keep_key(const KvEvictArgs& a, float w, uint32_t position, uint32_t next, bool crowded) {
  const bool safe = is_protected(a, position, next);
  if (safe != crowded) return safe ? 0xFFFFFFFFU : 0U;
  const uint32_t bits = w != w ? 0xFF800000U : __float_as_uint(w + 0.0F);
  return (bits & 0x80000000U) ? ~bits : bits | 0x80000000U;
}

// Ranks of two flags in thread order over the CTA, and their totals.
__device__ __forceinline__ void block_ranks(bool a, bool b, uint32_t* scratch, uint32_t* rank_a, uint32_t* rank_b,
                                            uint32_t* total_a, uint32_t* total_b) {
  const uint32_t lane = threadIdx.x & 31U, warp = threadIdx.x >> 5U;
  const uint32_t below = (1U << lane) - 1U;
  const uint32_t va = __ballot_sync(0xffffffffU, a), vb = __ballot_sync(0xffffffffU, b);
  __syncthreads();  // the scratch of the call before has been read
  if (lane == 0U) {
    scratch[warp] = __popc(va);
    scratch[32U + warp] = __popc(vb);
  }
  __syncthreads();
  uint32_t before_a = 0U, before_b = 0U, sum_a = 0U, sum_b = 0U;
  for (uint32_t w = 0; w < kSelectThreads / 32U; ++w) {
    const uint32_t ca = scratch[w], cb = scratch[32U + w];
    if (w < warp) { before_a += ca; before_b += cb; }
    sum_a += ca;
    sum_b += cb;
  }
  *rank_a = before_a + __popc(va & below);
  *rank_b = before_b + __popc(vb & below);
  *total_a = sum_a;
  *total_b = sum_b;
}

__global__ void __launch_bounds__(kSelectThreads) kv_select_kernel(KvEvictArgs a, RowHeader* headers, uint2* pairs, uint32_t most) {
  __shared__ uint32_t bins[256], scratch[64], chosen[2];
  const uint32_t s = blockIdx.y;
  const size_t row = static_cast<size_t>(s) * a.cache.kv_heads + blockIdx.x;
  const uint32_t n = min(a.lengths_in[s], kv_capacity(a.cache));
  const uint32_t m = min(n, a.budget);
  const uint32_t next = a.next_positions[s];
  const float* w = a.weights_in + row * a.stride;
  const uint32_t* pos = a.positions_in + row * a.stride;
  float* w_out = a.weights_out + row * a.stride;
  uint32_t* pos_out = a.positions_out + row * a.stride;
  uint32_t threshold = 0U, ties = n;  // n <= budget: everything is kept
  bool crowded = false;
  if (n > m) {
    uint32_t safe = 0U;
    for (uint32_t t0 = 0; t0 < n; t0 += kSelectThreads) {
      const uint32_t t = t0 + threadIdx.x;
      safe += __syncthreads_count(t < n && is_protected(a, pos[t], next));
    }
    crowded = safe > m;
    uint32_t left = m, prefix = 0U;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (threadIdx.x < 256U) bins[threadIdx.x] = 0U;
      __syncthreads();
      for (uint32_t t = threadIdx.x; t < n; t += kSelectThreads) {
        const uint32_t key = keep_key(a, w[t], pos[t], next, crowded);
        if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&bins[(key >> shift) & 255U], 1U);
      }
      __syncthreads();
      if (threadIdx.x == 0U) {
        uint32_t above = 0U, digit = 255U;
        while (above + bins[digit] < left) above += bins[digit--];
        chosen[0] = digit;
        chosen[1] = above;
      }
      __syncthreads();
      prefix = (prefix << 8U) | chosen[0];
      left -= chosen[1];
    }
    threshold = prefix;
    ties = left;
  }
  uint32_t tied = 0U, holes = 0U, movers = 0U;
  for (uint32_t t0 = 0; t0 < n; t0 += kSelectThreads) {
    const uint32_t t = t0 + threadIdx.x;
    const uint32_t key = t < n ? keep_key(a, w[t], pos[t], next, crowded) : 0U;
    const bool tie = t < n && n > m && key == threshold;
    uint32_t rank, rank2, total, total2;
    block_ranks(tie, false, scratch, &rank, &rank2, &total, &total2);
    const bool keep = t < n && (n == m || key > threshold || (tie && tied + rank < ties));
    tied += total;
    const bool hole = t < m && !keep, mover = t >= m && keep;
    block_ranks(hole, mover, scratch, &rank, &rank2, &total, &total2);
    if (hole && holes + rank < most) pairs[row * most + holes + rank].x = t;
    if (mover && movers + rank2 < most) pairs[row * most + movers + rank2].y = t;
    holes += total;
    movers += total2;
    if (t < m && keep) {
      if (w_out != w) w_out[t] = w[t];
      if (pos_out != pos) pos_out[t] = pos[t];
    }
    if (t >= m && t < n && !keep) w_out[t] = 0.0F;
  }
  if (threadIdx.x == 0U) headers[row] = {n, m, min(holes, most), 0U};
}

// grid (rows, chunks): one warp per move
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(KvEvictArgs a, const RowHeader* headers, const uint2* pairs, uint32_t most) {
  pdl_wait();
  const uint32_t row = blockIdx.x, s = row / a.cache.kv_heads, h = row % a.cache.kv_heads;
  const RowHeader header = headers[row];
  const uint32_t lane = threadIdx.x & 31U;
  if (h == 0U && blockIdx.y == 0U && threadIdx.x == 0U) a.lengths_out[s] = header.kept;
  const uint32_t pt = a.cache.page_tokens, hd = a.cache.head_dim;
  const uint32_t halves = a.cache.encoding == QLLM_KV_F16 ? hd : a.cache.encoding == QLLM_KV_Q8 ? hd / 2U + 1U : hd / 4U;
  for (uint32_t i = blockIdx.y * (kMoveThreads / 32U) + threadIdx.x / 32U; i < header.moves; i += gridDim.y * (kMoveThreads / 32U)) {
    const uint2 pair = pairs[static_cast<size_t>(row) * most + i];
    uint8_t* to = kv_page(a.cache, s, pair.x / pt);
    const uint8_t* from = kv_page(a.cache, s, pair.y / pt);
    if (to && from) {
#pragma unroll
      for (int value = 0; value < 2; ++value) {
        uint16_t* dst = reinterpret_cast<uint16_t*>(to + kv_codes_at(a.cache, value != 0, pair.x % pt, h));
        const uint16_t* src = reinterpret_cast<const uint16_t*>(from + kv_codes_at(a.cache, value != 0, pair.y % pt, h));
        for (uint32_t j = lane; j < halves; j += 32U) dst[j] = src[j];
        if (a.cache.encoding == QLLM_KV_Q4H && lane == 0U)
          *reinterpret_cast<uint16_t*>(to + kv_scale_at(a.cache, value != 0, pair.x % pt, h)) =
              *reinterpret_cast<const uint16_t*>(from + kv_scale_at(a.cache, value != 0, pair.y % pt, h));
      }
    }
    if (lane == 0U) {
      const size_t at = static_cast<size_t>(row) * a.stride;
      const float w = a.weights_in[at + pair.y];
      const uint32_t position = a.positions_in[at + pair.y];
      a.weights_out[at + pair.x] = w;
      a.positions_out[at + pair.x] = position;
      a.weights_out[at + pair.y] = 0.0F;
    }
  }
}

}  // namespace

size_t kv_evict_workspace_bytes(const KvBatch& c, uint32_t budget) {
  const size_t rows = static_cast<size_t>(c.sequences) * c.kv_heads;
  return rows * (sizeof(RowHeader) + static_cast<size_t>(most_moves(c, budget)) * sizeof(uint2));
}

int launch_kv_evict(const KvEvictArgs& a, cudaStream_t stream) {
  const uint32_t rows = a.cache.sequences * a.cache.kv_heads;
  const uint32_t most = most_moves(a.cache, a.budget);
  RowHeader* headers = static_cast<RowHeader*>(a.workspace);
  uint2* pairs = reinterpret_cast<uint2*>(headers + rows);
  kv_select_kernel<<<dim3(a.cache.kv_heads, a.cache.sequences), kSelectThreads, 0, stream>>>(a, headers, pairs, most);
  count_launch();
  const int rc = check_launch("kv_evict selection");
  if (rc) return rc;
  const uint32_t per_block = kMoveThreads / 32U;
  const uint32_t chunks = max(1U, min((most + per_block - 1U) / per_block, 64U));
  count_launch();
  return check_cuda(launch_pdl(kv_move_kernel, dim3(rows, chunks), dim3(kMoveThreads), 0, stream, a, headers, pairs, most), "kv_evict move");
}

}  // namespace qllm
