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

constexpr uint32_t kSelectThreads = 512;
constexpr uint32_t kSelectWarps = kSelectThreads / 32;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kSlotsPerBlock = 4096;  // a row is spread over more blocks only above this
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kAhead = 8;
constexpr uint32_t kMaxKeys = 48U * 1024U;  // of one block in shared memory; longer rows read weights and positions again
constexpr uint32_t kMoveThreads = 256;
constexpr uint32_t kMoveBatch = 64;       // moves

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

__global__ void __launch_bounds__(kSelectThreads, 2)
kv_select_kernel(const __grid_constant__ KvEvictArgs a, RowHeader* headers, uint2* pairs, uint32_t most, uint32_t keys_held) {
  extern __shared__ uint32_t keys[];
  __shared__ alignas(16) uint32_t bins[2][kBins];
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
  const auto barrier = [&] {
    if (blocks == 1U) __syncthreads();
    else cluster.sync();
  };
  const bool held = slice <= keys_held;
  bool crowded = false;
  const auto make_key = [&](uint32_t i) { return keep_key(a, w[first + i], pos[first + i], next, crowded); };
  const auto key_of = [&](uint32_t i) { return held ? keys[i] : make_key(i); };

  // the keys, kAhead loads of a thread in flight
  const uint32_t rounds = (count + kSelectThreads - 1U) / kSelectThreads;
  const auto make_keys = [&] {
    if (!held) return;
    for (uint32_t j = 0; j < rounds; j += kAhead) {
      float weight[kAhead];
      uint32_t position[kAhead];
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        const uint32_t i = (j + u) * kSelectThreads + tid;
        weight[u] = i < count ? w[first + i] : 0.0F;
        position[u] = i < count ? pos[first + i] : 0U;
      }
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        const uint32_t i = (j + u) * kSelectThreads + tid;
        if (i < count) keys[i] = keep_key(a, weight[u], position[u], next, crowded);
      }
    }
  };

  // ---- the m-th largest key
  uint32_t left = m, prefix = 0U, shift = 21U, buffer = 0U;
  for (uint32_t i = tid; i < kBins; i += kSelectThreads) bins[0][i] = 0U;
  make_keys();
  __syncthreads();
  for (;;) {
    const uint32_t top = shift + (shift == 0U ? 10U : 11U);  // bits from here on are the prefix
    for (uint32_t j = 0; j < rounds; j += 4U) {
      uint32_t four[4];
#pragma unroll
      for (uint32_t u = 0; u < 4U; ++u) {
        const uint32_t i = (j + u) * kSelectThreads + tid;
        four[u] = i < count ? key_of(i) : 0U;
      }
#pragma unroll
      for (uint32_t u = 0; u < 4U; ++u) {
        const uint32_t key = four[u];
        const bool counts_here = (j + u) * kSelectThreads + tid < count && (shift == 21U || (key >> top) == prefix);
        // the digit of the warp's first counting lane is added once for all lanes that share it: equal weights would
        // otherwise queue up at one address
        const uint32_t who = __ballot_sync(0xffffffffU, counts_here);
        if (who == 0U) continue;
        const uint32_t digit = (key >> shift) & (shift == 0U ? 1023U : 2047U);
        const uint32_t leader = __ffs(who) - 1U;
        const uint32_t common = __shfl_sync(0xffffffffU, digit, leader);
        const uint32_t same = __ballot_sync(0xffffffffU, counts_here && digit == common);
        if (lane == leader) atomicAdd(&bins[buffer][common], static_cast<uint32_t>(__popc(same)));
        else if (counts_here && digit != common) atomicAdd(&bins[buffer][digit], 1U);
      }
    }
    barrier();
    // thread t: bins 2047 - 4t down to 2044 - 4t of the whole cluster
    static_assert(kBins == 4U * kSelectThreads, "four bins to a thread");
    uint32_t v[4] = {0U, 0U, 0U, 0U};
    const uint32_t bin = kBins - 1U - 4U * tid;
    for (uint32_t b = 0; b < blocks; ++b) {
      const uint4 x = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&bins[buffer][bin - 3U], b));
      v[0] += x.w;
      v[1] += x.z;
      v[2] += x.y;
      v[3] += x.x;
    }
    // the other buffer was last read before the barrier above
    reinterpret_cast<uint4*>(bins[buffer ^ 1U])[tid] = make_uint4(0U, 0U, 0U, 0U);
    const uint32_t last_bin = v[0];  // thread 0: bin 2047
    const uint32_t own = v[0] + v[1] + v[2] + v[3];
    uint32_t upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffU, upto, o);
      if (lane >= static_cast<uint32_t>(o)) upto += t;
    }
    if (lane == 31U) warp_sums[warp] = upto;
    __syncthreads();
    uint32_t before = __reduce_add_sync(0xffffffffU, lane < warp ? warp_sums[lane] : 0U) + upto - own;
    if (before < left && left <= before + own) {
      uint32_t k = 0U;
      while (before + v[0] < left) {
        before += v[0];
        v[0] = v[1];
        v[1] = v[2];
        v[2] = v[3];
        ++k;
      }
      chosen[0] = bin - k;
      chosen[1] = before;
    }
    if (tid == 0U) chosen[2] = last_bin;
    __syncthreads();
    buffer ^= 1U;
    // the last bin of the first digit holds the protected slots alone (+infinity's key begins with another)
    if (shift == 21U && !crowded && chosen[2] > m) {
      crowded = true;
      make_keys();
      __syncthreads();
      continue;
    }
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
    const Counts v = lane < kSelectWarps ? warp_counts[lane] : Counts{};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      before.over[k] = __reduce_add_sync(0xffffffffU, lane < warp ? v.over[k] : 0U);
      before.tied[k] = __reduce_add_sync(0xffffffffU, lane < warp ? v.tied[k] : 0U);
      all.over[k] = __reduce_add_sync(0xffffffffU, v.over[k]);
      all.tied[k] = __reduce_add_sync(0xffffffffU, v.tied[k]);
    }
  }
  if (tid == 0U) counts = all;
  if (blocks > 1U) cluster.sync();
  // ties, kept slots below m and movers in the blocks before this one
  uint32_t ties_before = 0U, kept_before = 0U, movers_before = 0U;
  for (uint32_t b = 0; b < rank; ++b) {
    const Counts v = *cluster.map_shared_rank(&counts, b);
    const uint32_t kept_ties = min(v.tied[0], ties - min(ties, ties_before));
    kept_before += v.over[0] + kept_ties;
    movers_before += v.over[1] + min(v.tied[1], ties - min(ties, ties_before + v.tied[0]));
    ties_before += v.tied[0] + v.tied[1];
  }
  if (blocks > 1U) cluster.sync();  // nobody leaves while its counts are read
  // ... and in the warps before this one (a segment's ties all come after those of the segments before it)
  const uint32_t kept_ties = min(before.tied[0], ties - min(ties, ties_before));
  uint32_t kept = kept_before + before.over[0] + kept_ties;
  uint32_t movers = movers_before + before.over[1] + min(before.tied[1], ties - min(ties, ties_before + before.tied[0]));
  uint32_t tied_so_far = ties_before + before.tied[0] + before.tied[1];
  uint32_t holes = min(m, first + seg0) - kept;
  uint2* list = pairs + row * most;
  for (uint32_t i4 = seg0; i4 < seg1; i4 += 32U * kAhead) {
    // what stays below m is copied where the outputs are other arrays than the inputs
    float weight[kAhead];
    uint32_t position[kAhead];
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t i = i4 + 32U * u + lane, t = first + i;
      weight[u] = w_out != w && i < seg1 && t < m ? w[t] : 0.0F;
      position[u] = pos_out != pos && i < seg1 && t < m ? pos[t] : 0U;
    }
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t i = i4 + 32U * u + lane, t = first + i;
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
        if (w_out != w) w_out[t] = weight[u];
        if (pos_out != pos) pos_out[t] = position[u];
      }
      if (here && t >= m && !keep) w_out[t] = 0.0F;
    }
  }
  // the last warp of the last block has counted every mover
  if (rank == blocks - 1U && warp == kSelectWarps - 1U && lane == 0U) headers[row] = {n, m, min(movers, most), 0U};
}

// Words of one record, K and V: 16 bytes each (F16, Q4H and its 2-byte scale), or 4 (Q8, whose records are on
// 2-byte boundaries) and the two bytes left.
__host__ __device__ __forceinline__ uint32_t record_words(uint32_t encoding, uint32_t hd) {
  return 2U * (encoding == QLLM_KV_F16 ? hd / 8U : encoding == QLLM_KV_Q4H ? hd / 32U + 1U : hd / 4U + 1U);
}

// grid (rows, chunks).  Moves in batches: first a thread per move finds its two pages and moves weight and position, then
// all threads copy words, kAtOnce of them in flight each.
template <uint32_t ENC>
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const __grid_constant__ KvEvictArgs a, const RowHeader* headers,
                                                               const uint2* pairs, uint32_t most) {
  constexpr int kAtOnce = 4;
  __shared__ uint8_t* codes[2][kMoveBatch];   // K codes of target and source, null: no page
  __shared__ uint8_t* scales[2][ENC == QLLM_KV_Q4H ? kMoveBatch : 1];
  pdl_wait();
  const uint32_t row = blockIdx.x, s = row / a.cache.kv_heads, h = row % a.cache.kv_heads;
  const RowHeader header = headers[row];
  if (h == 0U && blockIdx.y == 0U && threadIdx.x == 0U) a.lengths_out[s] = header.kept;
  const uint32_t pt = a.cache.page_tokens, hd = a.cache.head_dim;
  const uint32_t words = record_words(ENC, hd), at_once = kMoveThreads / words;  // moves of a block side by side
  const uint32_t local = threadIdx.x / words, part = threadIdx.x % words;
  const bool value = part >= words / 2U;
  const uint32_t word = value ? part - words / 2U : part;
  const bool is_scale = ENC == QLLM_KV_Q4H && word == hd / 32U;
  // from a record's K codes (scale) to the thread's word
  const size_t to_value = value ? kv_codes_at(a.cache, true, 0U, 0U) : 0U;
  const size_t delta = to_value + (ENC == QLLM_KV_Q8 || is_scale ? 0U : 16U * word);
  const uint2* list = pairs + static_cast<size_t>(row) * most;
  const size_t at = static_cast<size_t>(row) * a.stride;
  for (uint32_t i0 = blockIdx.y * kMoveBatch; i0 < header.moves; i0 += gridDim.y * kMoveBatch) {
    const uint32_t count = min(kMoveBatch, header.moves - i0);
    __syncthreads();  // the batch before has been copied
    if (threadIdx.x < 2U * kMoveBatch) {
      const uint32_t i = threadIdx.x % kMoveBatch, side = threadIdx.x / kMoveBatch;
      if (i < count) {
        const uint2 pair = list[i0 + i];
        const uint32_t slot = side ? pair.y : pair.x, page = slot / pt, place = slot - page * pt;
        uint8_t* layer = kv_page(a.cache, s, page);
        codes[side][i] = layer ? layer + kv_codes_at(a.cache, false, place, h) : nullptr;
        if constexpr (ENC == QLLM_KV_Q4H) scales[side][i] = layer ? layer + kv_scale_at(a.cache, false, place, h) : nullptr;
        if (side) {
          const float w = a.weights_in[at + pair.y];
          const uint32_t position = a.positions_in[at + pair.y];
          a.weights_out[at + pair.x] = w;
          a.positions_out[at + pair.x] = position;
          a.weights_out[at + pair.y] = 0.0F;
        }
      }
    }
    __syncthreads();
    if (local >= at_once) continue;
    for (uint32_t j0 = local; j0 < count; j0 += kAtOnce * at_once) {
      uint8_t* to[kAtOnce];
      uint4 data[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const uint32_t j = j0 + u * at_once;
        to[u] = nullptr;
        data[u] = make_uint4(0U, 0U, 0U, 0U);
        if (j >= count || !codes[0][j] || !codes[1][j]) continue;
        if constexpr (ENC == QLLM_KV_Q8) {
          // hd + 2 bytes: whole words from the target's first 4-byte boundary on, and the two bytes before or behind them
          to[u] = codes[0][j] + delta;
          const uint8_t* from = codes[1][j] + delta;
          const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to[u])) & 2U;
          const uint32_t offset = word < hd / 4U ? odd + 4U * word : odd ? 0U : hd;
          to[u] += offset;
          const uint8_t* p = from + offset;
          if (word < hd / 4U && (reinterpret_cast<uintptr_t>(p) & 2U) == 0U) data[u].x = *reinterpret_cast<const uint32_t*>(p);
          else {
            data[u].x = *reinterpret_cast<const uint16_t*>(p);
            if (word < hd / 4U) data[u].x |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + 2)) << 16U;
          }
        } else if (is_scale) {
          to[u] = scales[0][ENC == QLLM_KV_Q4H ? j : 0U] + delta;
          data[u].x = *reinterpret_cast<const uint16_t*>(scales[1][ENC == QLLM_KV_Q4H ? j : 0U] + delta);
        } else {
          to[u] = codes[0][j] + delta;
          data[u] = *reinterpret_cast<const uint4*>(codes[1][j] + delta);
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (!to[u]) continue;
        if (ENC == QLLM_KV_Q8 ? word == hd / 4U : is_scale) *reinterpret_cast<uint16_t*>(to[u]) = static_cast<uint16_t>(data[u].x);
        else if (ENC == QLLM_KV_Q8) *reinterpret_cast<uint32_t*>(to[u]) = data[u].x;
        else *reinterpret_cast<uint4*>(to[u]) = data[u];
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

  // blocks per row: as many as fill the GPU, but only for rows of more than kSlotsPerBlock slots a block (a cluster's
  // barriers cost more than a short walk); and as many as it takes to hold the keys
  int device = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return check_cuda(e, "kv_evict device");
  const uint32_t capacity = kv_capacity(a.cache);
  uint32_t cluster = 1U;
  while (cluster < kMaxCluster && ((rows * cluster < static_cast<uint32_t>(sms) && capacity / cluster > kSlotsPerBlock) ||
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

  // a block per batch, up to 32 blocks per multiprocessor (8: 143 us, 32: 133 us, 64: 133 us for 8 x 8 rows of 8455 moves: rows
  // that move less leave room to the others)
  const uint32_t wanted = (most + kMoveBatch - 1U) / kMoveBatch, room = 32U * static_cast<uint32_t>(sms) / rows;
  const uint32_t chunks = max(1U, min(wanted, room));
  count_launch();
  const dim3 grid(rows, chunks), block(kMoveThreads);
  if (a.cache.encoding == QLLM_KV_F16) e = launch_pdl(kv_move_kernel<QLLM_KV_F16>, grid, block, 0, stream, a, headers, pairs, most);
  else if (a.cache.encoding == QLLM_KV_Q4H) e = launch_pdl(kv_move_kernel<QLLM_KV_Q4H>, grid, block, 0, stream, a, headers, pairs, most);
  else e = launch_pdl(kv_move_kernel<QLLM_KV_Q8>, grid, block, 0, stream, a, headers, pairs, most);
  return check_cuda(e, "kv_evict move");
}

}  // namespace qllm
