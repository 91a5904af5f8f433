// Eviction from the paged cache by accumulated attention weight (qllm_k_kv_evict).
//
// Per (sequence, kv head) of n slots, m = min(n, budget) are kept: first the protected ones (position
// among the last `recent` or the first `sinks`), then by weight, ties to the lower slot.  Kept slots
// below m stay where they are; the i-th freed slot below m takes the i-th kept slot at or above m.
// Sources and targets are disjoint, so the move is in place without an order between its copies,
// and no more than min(m, n - m) records move.
//
// First launch: selection.  The order is that of a 32-bit key, and the m-th largest key is found by three
// histograms of its digits (11, 11 and 10 bits) instead of a sort; then the slots are walked in order for
// the ties and for the ranks of the freed and the moving slots.  One cluster of blocks per (sequence, kv head): the
// keys are computed once and stay in shared memory (4 bytes a slot), and a histogram is summed over the cluster's blocks
// through distributed shared memory, so that a few long rows use the whole GPU.  Latency-bound: 8 bytes a
// slot are read once; the rest is a chain of some ten block and cluster barriers.
// Second launch: the moves, HBM-bound.
#include <cooperative_groups.h>

#include "kv_batch.cuh"
#include "launch.cuh"

namespace cg = cooperative_groups;

namespace qllm {

namespace {

constexpr uint32_t kSelectThreads = 1024;
constexpr uint32_t kSelectWarps = kSelectThreads / 32;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kMaxKeys = 48U * 1024U;  // of one block in shared memory; longer rows read weights and positions again
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

// What the slots of one block (or warp) hold, below and at or above m.
struct Counts {
  uint32_t over[2], tied[2];  // keys above the threshold, keys equal to it
};

__global__ void __launch_bounds__(kSelectThreads, 1)
kv_select_kernel(const __grid_constant__ KvEvictArgs a, RowHeader* headers, uint2* pairs, uint32_t most, uint32_t keys_held) {
  extern __shared__ uint32_t keys[];
  __shared__ alignas(8) uint32_t bins[2][kBins];
  __shared__ uint32_t warp_sums[kSelectWarps], chosen[3];
  __shared__ Counts warp_counts[kSelectWarps], counts;
  const cg::cluster_group cluster = cg::this_cluster();
  const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const size_t row = blockIdx.x / blocks;
  const uint32_t s = static_cast<uint32_t>(row / a.cache.kv_heads);
  const uint32_t tid = threadIdx.x, lane = tid & 31U, warp = tid >> 5U, below = (1U << lane) - 1U;
  const uint32_t n = min(a.lengths_in[s], kv_capacity(a.cache));
  const uint32_t m = min(n, a.budget);
  const uint32_t next = a.next_positions[s];
  const float* w = a.weights_in + row * a.stride;
  const uint32_t* pos = a.positions_in + row * a.stride;
  float* w_out = a.weights_out + row * a.stride;
  uint32_t* pos_out = a.positions_out + row * a.stride;
  // this block's slots [first, first + count)
  const uint32_t slice = ((n + blocks - 1U) / blocks + 31U) & ~31U;
  const uint32_t first = min(n, rank * slice), count = min(slice, n - first);
  if (n == m) {  // everything stays; the whole cluster leaves
    for (uint32_t t = first + tid; t < first + count; t += kSelectThreads) {
      if (w_out != w) w_out[t] = w[t];
      if (pos_out != pos) pos_out[t] = pos[t];
    }
    if (rank == 0U && tid == 0U) headers[row] = {n, m, 0U, 0U};
    return;
  }
  const bool held = slice <= keys_held;
  bool crowded = false;
  const auto make_key = [&](uint32_t i) { return keep_key(a, w[first + i], pos[first + i], next, crowded); };
  const auto key_of = [&](uint32_t i) { return held ? keys[i] : make_key(i); };

  // ---- the m-th largest key
  uint32_t left = m, prefix = 0U, shift = 21U, buffer = 0U;
  for (uint32_t i = tid; i < kBins; i += kSelectThreads) bins[0][i] = 0U;
  bool fresh = true;  // the keys are to be made
  __syncthreads();
  for (;;) {
    const uint32_t rounds = (count + kSelectThreads - 1U) / kSelectThreads;
    const uint32_t top = shift + (shift == 0U ? 10U : 11U);  // bits from here on are the prefix
#pragma unroll 4
    for (uint32_t j = 0; j < rounds; ++j) {
      const uint32_t i = j * kSelectThreads + tid;
      uint32_t key = 0U;
      if (i < count) {
        if (fresh) {
          key = make_key(i);
          if (held) keys[i] = key;
        } else {
          key = key_of(i);
        }
      }
      const bool counts_here = i < count && (shift == 21U || (key >> top) == prefix);
      const uint32_t digit = (key >> shift) & (shift == 0U ? 1023U : 2047U);
      // the digit of the warp's first counting lane is added once for all lanes that share it: equal weights would
      // otherwise queue up at one address
      const uint32_t who = __ballot_sync(0xffffffffU, counts_here);
      if (who == 0U) continue;
      const uint32_t leader = __ffs(who) - 1U;
      const uint32_t common = __shfl_sync(0xffffffffU, digit, leader);
      const uint32_t same = __ballot_sync(0xffffffffU, counts_here && digit == common);
      if (lane == leader) atomicAdd(&bins[buffer][common], static_cast<uint32_t>(__popc(same)));
      else if (counts_here && digit != common) atomicAdd(&bins[buffer][digit], 1U);
    }
    cluster.sync();
    // thread t: bins 2047 - 2t and 2046 - 2t of the whole cluster, in descending order
    uint32_t high = 0U, low = 0U;
    const uint32_t bin = kBins - 1U - 2U * tid;
    for (uint32_t b = 0; b < blocks; ++b) {
      const uint2 v = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&bins[buffer][bin - 1U], b));
      low += v.x;
      high += v.y;
    }
    // the other buffer was last read before the barrier above
    reinterpret_cast<uint2*>(bins[buffer ^ 1U])[tid] = make_uint2(0U, 0U);
    uint32_t upto = high + low;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffU, upto, o);
      if (lane >= static_cast<uint32_t>(o)) upto += t;
    }
    if (lane == 31U) warp_sums[warp] = upto;
    __syncthreads();
    uint32_t before = warp_sums[lane];
    before = __reduce_add_sync(0xffffffffU, lane < warp ? before : 0U) + upto - high - low;
    if (before < left && left <= before + high + low) {
      const bool in_high = left <= before + high;
      chosen[0] = in_high ? bin : bin - 1U;
      chosen[1] = in_high ? before : before + high;
    }
    if (tid == 0U) chosen[2] = high;
    __syncthreads();
    buffer ^= 1U;
    // the last bin of the first digit holds the protected slots alone (+infinity's key begins with another)
    if (shift == 21U && !crowded && chosen[2] > m) {
      crowded = true;
      fresh = true;
      __syncthreads();
      continue;
    }
    fresh = false;
    prefix = (prefix << (shift == 0U ? 10U : 11U)) | chosen[0];
    left -= chosen[1];
    if (shift == 0U) break;
    shift = shift == 21U ? 10U : 0U;
    __syncthreads();  // `chosen` has been read
  }
  const uint32_t threshold = prefix, ties = left;  // the first `ties` slots of that key are kept

  // ---- ranks.  Each warp walks a contiguous segment of the block's slots.
  const uint32_t segment = ((count + kSelectWarps - 1U) / kSelectWarps + 31U) & ~31U;
  const uint32_t seg0 = min(count, warp * segment), seg1 = min(count, seg0 + segment);
  Counts mine{};
  for (uint32_t i0 = seg0; i0 < seg1; i0 += 32U) {
    const uint32_t i = i0 + lane;
    const uint32_t key = i < seg1 ? key_of(i) : 0U;
    const uint32_t over = __ballot_sync(0xffffffffU, i < seg1 && key > threshold);
    const uint32_t tied = __ballot_sync(0xffffffffU, i < seg1 && key == threshold);
    // lanes whose slot lies below m
    const uint32_t under = first + i0 >= m ? 0U : m - first - i0 >= 32U ? 0xffffffffU : (1U << (m - first - i0)) - 1U;
    mine.over[0] += __popc(over & under);
    mine.over[1] += __popc(over & ~under);
    mine.tied[0] += __popc(tied & under);
    mine.tied[1] += __popc(tied & ~under);
  }
  if (lane == 0U) warp_counts[warp] = mine;
  __syncthreads();
  // sums over the warps before this one, and over all of them
  Counts before{}, all{};
  {
    const Counts v = warp_counts[lane];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      before.over[k] = __reduce_add_sync(0xffffffffU, lane < warp ? v.over[k] : 0U);
      before.tied[k] = __reduce_add_sync(0xffffffffU, lane < warp ? v.tied[k] : 0U);
      all.over[k] = __reduce_add_sync(0xffffffffU, v.over[k]);
      all.tied[k] = __reduce_add_sync(0xffffffffU, v.tied[k]);
    }
  }
  if (tid == 0U) counts = all;
  cluster.sync();
  // ties, kept slots below m and movers in the blocks before this one
  uint32_t ties_before = 0U, kept_before = 0U, movers_before = 0U;
  for (uint32_t b = 0; b < rank; ++b) {
    const Counts v = *cluster.map_shared_rank(&counts, b);
    const uint32_t kept_ties = min(v.tied[0], ties - min(ties, ties_before));
    kept_before += v.over[0] + kept_ties;
    movers_before += v.over[1] + min(v.tied[1], ties - min(ties, ties_before + v.tied[0]));
    ties_before += v.tied[0] + v.tied[1];
  }
  cluster.sync();  // nobody leaves while its counts are read
  // ... and in the warps before this one (a segment's ties all come after those of the segments before it)
  const uint32_t kept_ties = min(before.tied[0], ties - min(ties, ties_before));
  uint32_t kept = kept_before + before.over[0] + kept_ties;
  uint32_t movers = movers_before + before.over[1] + min(before.tied[1], ties - min(ties, ties_before + before.tied[0]));
  uint32_t tied_so_far = ties_before + before.tied[0] + before.tied[1];
  uint32_t holes = min(m, first + seg0) - kept;
  uint2* list = pairs + row * most;
  for (uint32_t i0 = seg0; i0 < seg1; i0 += 32U) {
    const uint32_t i = i0 + lane, t = first + i;
    const bool here = i < seg1;
    const uint32_t key = here ? key_of(i) : 0U;
    const uint32_t tied = __ballot_sync(0xffffffffU, here && key == threshold);
    const bool keep = here && (key > threshold || (key == threshold && tied_so_far + __popc(tied & below) < ties));
    tied_so_far += __popc(tied);
    const bool hole = here && t < m && !keep, mover = here && t >= m && keep;
    const uint32_t hole_mask = __ballot_sync(0xffffffffU, hole), mover_mask = __ballot_sync(0xffffffffU, mover);
    const uint32_t hole_rank = holes + __popc(hole_mask & below), mover_rank = movers + __popc(mover_mask & below);
    if (hole && hole_rank < most) list[hole_rank].x = t;
    if (mover && mover_rank < most) list[mover_rank].y = t;
    holes += __popc(hole_mask);
    movers += __popc(mover_mask);
    if (here && t < m && keep) {
      if (w_out != w) w_out[t] = w[t];
      if (pos_out != pos) pos_out[t] = pos[t];
    }
    if (here && t >= m && !keep) w_out[t] = 0.0F;
  }
  // the last warp of the last block has counted every mover
  if (rank == blocks - 1U && warp == kSelectWarps - 1U && lane == 0U) headers[row] = {n, m, min(movers, most), 0U};
}

// Words of one record, K and V: 16 bytes each (F16, Q4H and its 2-byte scale), or 4 (Q8, whose records are on
// 2-byte boundaries) and the two bytes left.
__host__ __device__ __forceinline__ uint32_t record_words(uint32_t encoding, uint32_t hd) {
  return 2U * (encoding == QLLM_KV_F16 ? hd / 8U : encoding == QLLM_KV_Q4H ? hd / 32U + 1U : hd / 4U + 1U);
}

// grid (rows, chunks).  A thread copies the same word of one record after another, kAtOnce of them in flight (a move is
// a chain of three loads: the pair, the page, the record).
template <uint32_t ENC>
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const __grid_constant__ KvEvictArgs a, const RowHeader* headers,
                                                               const uint2* pairs, uint32_t most) {
  constexpr int kAtOnce = 4;
  pdl_wait();
  const uint32_t row = blockIdx.x, s = row / a.cache.kv_heads, h = row % a.cache.kv_heads;
  const RowHeader header = headers[row];
  if (h == 0U && blockIdx.y == 0U && threadIdx.x == 0U) a.lengths_out[s] = header.kept;
  const uint32_t pt = a.cache.page_tokens, hd = a.cache.head_dim;
  const uint32_t words = record_words(ENC, hd), at_once = kMoveThreads / words;  // moves of a block side by side
  const uint32_t local = threadIdx.x / words, part = threadIdx.x % words;
  if (local >= at_once) return;
  const bool value = part >= words / 2U;
  const uint32_t word = value ? part - words / 2U : part;
  const bool is_scale = ENC == QLLM_KV_Q4H && word == hd / 32U;
  const uint2* list = pairs + static_cast<size_t>(row) * most;
  const size_t at = static_cast<size_t>(row) * a.stride;
  const uint32_t step = gridDim.y * at_once;
  // where the thread's word of the record of a slot lies; null without a page
  const auto find = [&](uint32_t slot, size_t* record) -> uint8_t* {
    const uint32_t page = slot / pt, place = slot - page * pt;
    uint8_t* layer = kv_page(a.cache, s, page);
    *record = is_scale ? kv_scale_at(a.cache, value, place, h) : kv_codes_at(a.cache, value, place, h) + (ENC == QLLM_KV_Q8 ? 0U : 16U * word);
    return layer ? layer + *record : nullptr;
  };
  for (uint32_t i0 = blockIdx.y * at_once + local; i0 < header.moves; i0 += kAtOnce * step) {
    uint2 pair[kAtOnce];
    uint8_t* to[kAtOnce];
    uint4 data[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) pair[u] = i0 + u * step < header.moves ? list[i0 + u * step] : make_uint2(kPaddingSlot, 0U);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      to[u] = nullptr;
      data[u] = make_uint4(0U, 0U, 0U, 0U);
      if (pair[u].x == kPaddingSlot) continue;
      size_t dst, src;
      to[u] = find(pair[u].x, &dst);
      const uint8_t* from = find(pair[u].y, &src);
      if (!from) to[u] = nullptr;
      if (!to[u]) continue;
      if constexpr (ENC == QLLM_KV_Q8) {
        // hd + 2 bytes: whole words from the target's first 4-byte boundary on, and the two bytes before or behind them
        const uint32_t odd = static_cast<uint32_t>(dst) & 2U;
        const uint32_t offset = word < hd / 4U ? odd + 4U * word : odd ? 0U : hd;
        to[u] += offset;
        const uint8_t* p = from + offset;
        if (word < hd / 4U && (static_cast<uint32_t>(src) & 2U) == odd) data[u].x = *reinterpret_cast<const uint32_t*>(p);
        else {
          data[u].x = *reinterpret_cast<const uint16_t*>(p);
          if (word < hd / 4U) data[u].x |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + 2)) << 16U;
        }
      } else if (is_scale) {
        data[u].x = *reinterpret_cast<const uint16_t*>(from);
      } else {
        data[u] = *reinterpret_cast<const uint4*>(from);
      }
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (to[u]) {
        if (ENC == QLLM_KV_Q8 ? word == hd / 4U : is_scale) *reinterpret_cast<uint16_t*>(to[u]) = static_cast<uint16_t>(data[u].x);
        else if (ENC == QLLM_KV_Q8) *reinterpret_cast<uint32_t*>(to[u]) = data[u].x;
        else *reinterpret_cast<uint4*>(to[u]) = data[u];
      }
      if (part == 0U && pair[u].x != kPaddingSlot) {
        const float w = a.weights_in[at + pair[u].y];
        const uint32_t position = a.positions_in[at + pair[u].y];
        a.weights_out[at + pair[u].x] = w;
        a.positions_out[at + pair[u].x] = position;
        a.weights_out[at + pair[u].y] = 0.0F;
      }
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

  // blocks per row: enough to fill the GPU, but not fewer than a slot per thread; and as many as it takes to hold the keys
  int device = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return check_cuda(e, "kv_evict device");
  const uint32_t capacity = kv_capacity(a.cache);
  uint32_t cluster = 1U;
  while (cluster < kMaxCluster && ((rows * cluster < static_cast<uint32_t>(sms) && capacity / cluster > kSelectThreads) ||
                                   capacity / cluster > kMaxKeys))
    cluster *= 2U;
  const uint32_t slice = ((capacity + cluster - 1U) / cluster + 31U) & ~31U;
  const uint32_t keys_held = min(slice, kMaxKeys);
  e = cudaFuncSetAttribute(kv_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxKeys * sizeof(uint32_t));
  if (e != cudaSuccess) return check_cuda(e, "kv_evict shared memory opt-in");
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(rows * cluster);
  config.blockDim = dim3(kSelectThreads);
  config.dynamicSmemBytes = keys_held * sizeof(uint32_t);
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = cluster;
  attribute.val.clusterDim.y = 1;
  attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  count_launch();
  const int rc = check_cuda(cudaLaunchKernelEx(&config, kv_select_kernel, a, headers, pairs, most, keys_held), "kv_evict selection");
  if (rc) return rc;

  // a thread per word of the largest move, up to eight blocks per multiprocessor
  const uint32_t per_block = kMoveThreads / record_words(a.cache.encoding, a.cache.head_dim);
  const uint32_t wanted = (most + per_block - 1U) / per_block, room = (8U * static_cast<uint32_t>(sms) + rows - 1U) / rows;
  const uint32_t chunks = max(1U, min(wanted, room));
  count_launch();
  const dim3 grid(rows, chunks), block(kMoveThreads);
  if (a.cache.encoding == QLLM_KV_F16) e = launch_pdl(kv_move_kernel<QLLM_KV_F16>, grid, block, 0, stream, a, headers, pairs, most);
  else if (a.cache.encoding == QLLM_KV_Q4H) e = launch_pdl(kv_move_kernel<QLLM_KV_Q4H>, grid, block, 0, stream, a, headers, pairs, most);
  else e = launch_pdl(kv_move_kernel<QLLM_KV_Q8>, grid, block, 0, stream, a, headers, pairs, most);
  return check_cuda(e, "kv_evict move");
}

}  // namespace qllm
