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
//
// Measured on one B200 (copy 6554 GB/s): 8 sequences of 32768 slots to half, F16, 8 kv heads of 128: 132 us, of which the
// selection takes 32 (issue: histogram atomics and the rank walks) and the moves 100 (540 MB, 0.83 of the copy rate); 48 of up to
// 6001 to 4096, Q4H, 4 heads of 128: 24 us (selection 18: its chain of barriers; moves of 66 bytes 6 to 12); one slot of 4097,
// 8 heads of 128: 11.6 us, latency alone.
#include <cooperative_groups.h>

#include "kv_batch.cuh"
#include "launch.cuh"

namespace cg = cooperative_groups;

namespace qllm {

namespace {

constexpr uint32_t kSelectThreads = 512;
constexpr uint32_t kSelectWarps = kSelectThreads / 32;
constexpr uint32_t kBins = 2048;
// A row is spread over more blocks only above this (2048 / 4096 / 8192, 8 heads of 128: 1 of 4097 11.3 / 11.6 / 12.1 us, 1 of 8192 to half
// 16.7 / 18.5 / 21.5, 4 of 8192 25.5 / 26.4 / 30.0, 1 of 16384 Q4H 20.1 / 19.0 / 23.4; 8 of 32768 and 48 of 6001 do not depend on it).
constexpr uint32_t kSlotsPerBlock = 4096;
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kAhead = 8;
constexpr uint32_t kMaxKeys = 48U * 1024U;  // of one block in shared memory; longer rows read weights and positions again
constexpr uint32_t kKeysByDefault = 7U * 1024U;  // that a launch may hold beside the static arrays without asking for more
constexpr uint32_t kMoveThreads = 256;
constexpr uint32_t kMoveBatch = 64;       // moves (32: 142 us, 64: 135 us, 128: 136 us for 8 x 8 rows of 8455)
constexpr uint32_t kMoveBlocks = 5;       // per multiprocessor, all of them at once

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
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ alignas(16) uint32_t bins[2][kBins];
  __shared__ uint32_t warp_sums[kSelectWarps], chosen[4];
  __shared__ Counts warp_counts[kSelectWarps], counts;
  const cg::cluster_group cluster = cg::this_cluster();
  const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const size_t row = blockIdx.x / blocks;
  const uint32_t s = static_cast<uint32_t>(row / a.cache.kv_heads);
  const uint32_t tid = threadIdx.x, lane = tid & 31U, warp = tid >> 5U;
  const uint32_t n = min(a.lengths_in[s], kv_capacity(a.cache));
  const uint32_t m = min(n, a.budget);
  const uint32_t next = a.next_positions[s];
  const float* w = a.weights_in + row * a.stride;
  const uint32_t* pos = a.positions_in + row * a.stride;
  float* w_out = a.weights_out + row * a.stride;
  uint32_t* pos_out = a.positions_out + row * a.stride;
  // this block's slots [first, first + count), in quads: a thread takes four neighbours at a time
  const uint32_t slice = ((n + blocks - 1U) / blocks + 127U) & ~127U;
  const uint32_t first = min(n, rank * slice), count = min(slice, n - first), quads = (count + 3U) / 4U;
  const bool held = slice <= keys_held;
  bool crowded = false;
  // One key into the histogram `to`, by all lanes of a warp.
  const auto count_key = [&](uint32_t* to, bool counts_here, uint32_t digit) {
    const uint32_t who = __ballot_sync(0xffffffffU, counts_here);
    if (__popc(who) >= 8) {
      // the digit of the warp's first counting lane is added once for all lanes that share it: equal weights would
      // otherwise queue up at one address
      const uint32_t leader = __ffs(who) - 1U;
      const uint32_t common = __shfl_sync(0xffffffffU, digit, leader);
      const uint32_t same = __ballot_sync(0xffffffffU, counts_here && digit == common);
      if (lane == leader) atomicAdd(&to[common], static_cast<uint32_t>(__popc(same)));
      else if (counts_here && digit != common) atomicAdd(&to[digit], 1U);
    } else if (counts_here) {
      atomicAdd(&to[digit], 1U);
    }
  };
  uint32_t buffer = 0U;
  // The keys, kAhead loads of a thread in flight, and (of keys that are held) the histogram of their first digit while other
  // warps wait for theirs.  Where the outputs are other arrays, they get what would be there without a move: the slots
  // below m as they are, zero weights behind.
  const auto make_keys = [&] {
    for (uint32_t j = 0; j < count; j += kAhead * kSelectThreads) {
      float weight[kAhead];
      uint32_t position[kAhead];
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        const uint32_t i = j + u * kSelectThreads + tid;
        weight[u] = i < count ? w[first + i] : 0.0F;
        position[u] = i < count ? pos[first + i] : 0U;
      }
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        const uint32_t i = j + u * kSelectThreads + tid, t = first + i;
        if (j + u * kSelectThreads >= count) break;
        if (held && n > m) {
          const uint32_t key = keep_key(a, weight[u], position[u], next, crowded);
          if (i < count) keys[i] = key;
          count_key(bins[buffer], i < count, key >> 21U);
        }
        if (i >= count) continue;
        if (w_out != w) w_out[t] = t < m ? weight[u] : 0.0F;
        if (pos_out != pos && t < m) pos_out[t] = position[u];
      }
    }
  };
  for (uint32_t i = tid; i < kBins; i += kSelectThreads) bins[0][i] = 0U;
  __syncthreads();
  make_keys();
  if (n == m) {  // everything stays; the whole cluster leaves
    if (rank == 0U && tid == 0U) headers[row] = {n, m, 0U, 0U};
    return;
  }
  const auto barrier = [&] {
    if (blocks == 1U) __syncthreads();
    else cluster.sync();
  };
  const auto four_keys = [&](uint32_t quad, uint32_t (&key)[4]) {
    if (held) {
      const uint4 v = reinterpret_cast<const uint4*>(keys)[quad];
      key[0] = v.x;
      key[1] = v.y;
      key[2] = v.z;
      key[3] = v.w;
    } else {
#pragma unroll
      for (uint32_t u = 0; u < 4U; ++u) {
        const uint32_t i = 4U * quad + u;
        key[u] = i < count ? keep_key(a, w[first + i], pos[first + i], next, crowded) : 0U;
      }
    }
  };

  // ---- the m-th largest key
  uint32_t threshold = 0U, ties = 0U;  // kept: keys above the threshold, and the first `ties` slots of that key
  uint32_t left = m, prefix = 0U, shift = 21U;
  const uint32_t rounds = (quads + kSelectThreads - 1U) / kSelectThreads;
  for (;;) {
    const uint32_t top = shift + (shift == 0U ? 10U : 11U);  // bits from here on are the prefix
    for (uint32_t j = 0; j < rounds; ++j) {
      if (held && shift == 21U) break;  // counted
      const uint32_t quad = j * kSelectThreads + tid;
      uint32_t four[4] = {0U, 0U, 0U, 0U};
      if (quad < quads) four_keys(quad, four);
#pragma unroll
      for (uint32_t u = 0; u < 4U; ++u)
        count_key(bins[buffer], 4U * quad + u < count && (shift == 21U || (four[u] >> top) == prefix),
                  (four[u] >> shift) & (shift == 0U ? 1023U : 2047U));
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
      chosen[3] = v[0];
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
    if (left == chosen[3] && prefix != 0U) {  // the cut falls between two bins: every key of this one is kept (a cache that
      threshold = (prefix << shift) - 1U;     // evicts a slot a step is done after one digit most of the time)
      break;
    }
    if (shift == 0U) {
      threshold = prefix;
      ties = left;
      break;
    }
    shift = shift == 21U ? 10U : 0U;
    __syncthreads();  // `chosen` has been read
  }

  // ---- ranks.  Each warp walks a contiguous segment of the block's quads.
  const uint32_t segment = ((quads + kSelectWarps - 1U) / kSelectWarps + 31U) & ~31U;
  const uint32_t seg0 = min(quads, warp * segment), seg1 = min(quads, seg0 + segment);
  Counts mine{};
  for (uint32_t q0 = seg0; q0 < seg1; q0 += 32U) {
    const uint32_t quad = q0 + lane;
    if (quad >= seg1) continue;
    uint32_t key[4];
    four_keys(quad, key);
#pragma unroll
    for (uint32_t u = 0; u < 4U; ++u) {
      const uint32_t i = 4U * quad + u, side = first + i < m ? 0U : 1U;
      const uint32_t over = i < count && key[u] > threshold ? 1U : 0U, tied = i < count && key[u] == threshold ? 1U : 0U;
      mine.over[0] += side ? 0U : over;
      mine.over[1] += side ? over : 0U;
      mine.tied[0] += side ? 0U : tied;
      mine.tied[1] += side ? tied : 0U;
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    mine.over[k] = __reduce_add_sync(0xffffffffU, mine.over[k]);
    mine.tied[k] = __reduce_add_sync(0xffffffffU, mine.tied[k]);
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
  // ties, kept slots below m and movers in the blocks before this one
  uint32_t ties_before = 0U, kept_before = 0U, movers_before = 0U;
  if (blocks > 1U) {
    if (tid == 0U) counts = all;
    cluster.sync();
    for (uint32_t b = 0; b < rank; ++b) {
      const Counts v = *cluster.map_shared_rank(&counts, b);
      kept_before += v.over[0] + min(v.tied[0], ties - min(ties, ties_before));
      movers_before += v.over[1] + min(v.tied[1], ties - min(ties, ties_before + v.tied[0]));
      ties_before += v.tied[0] + v.tied[1];
    }
    cluster.sync();  // nobody leaves while its counts are read
  }
  // ... and in the warps before this one (a segment's ties all come after those of the segments before it)
  const uint32_t kept = kept_before + before.over[0] + min(before.tied[0], ties - min(ties, ties_before));
  uint32_t movers = movers_before + before.over[1] + min(before.tied[1], ties - min(ties, ties_before + before.tied[0]));
  uint32_t tied_so_far = ties_before + before.tied[0] + before.tied[1];
  uint32_t holes = min(m, first + 4U * seg0) - kept;
  uint2* list = pairs + row * most;
  for (uint32_t q0 = seg0; q0 < seg1; q0 += 32U) {
    const uint32_t quad = q0 + lane;
    uint32_t key[4] = {0U, 0U, 0U, 0U};
    if (quad < seg1) four_keys(quad, key);
    uint32_t tied = 0U, inside = 0U;  // bit u: the lane's slot u counts
#pragma unroll
    for (uint32_t u = 0; u < 4U; ++u) {
      if (quad < seg1 && 4U * quad + u < count) inside |= 1U << u;
      if (key[u] == threshold) tied |= 1U << u;
    }
    tied &= inside;
    uint32_t tie = tied_so_far;  // rank of the lane's first tie
    if (__any_sync(0xffffffffU, tied != 0U)) {
      uint32_t upto = __popc(tied);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffU, upto, o);
        if (lane >= static_cast<uint32_t>(o)) upto += t;
      }
      tie += upto - __popc(tied);
      tied_so_far += __shfl_sync(0xffffffffU, upto, 31);
    }
    uint32_t hole = 0U, mover = 0U;
#pragma unroll
    for (uint32_t u = 0; u < 4U; ++u) {
      const uint32_t t = first + 4U * quad + u;
      const bool keep = key[u] > threshold || ((tied >> u & 1U) && tie < ties);
      tie += tied >> u & 1U;
      if (!(inside >> u & 1U)) continue;
      if (t < m) {
        if (!keep) hole |= 1U << u;
      } else if (keep) {
        mover |= 1U << u;
      } else if (w_out == w) {
        w_out[t] = 0.0F;
      }
    }
    if (!__any_sync(0xffffffffU, (hole | mover) != 0U)) continue;
    const uint32_t both = __popc(hole) | __popc(mover) << 16U;  // at most 128 of each
    uint32_t upto = both;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffU, upto, o);
      if (lane >= static_cast<uint32_t>(o)) upto += t;
    }
    uint32_t hole_rank = holes + ((upto - both) & 0xffffU), mover_rank = movers + ((upto - both) >> 16U);
#pragma unroll
    for (uint32_t u = 0; u < 4U; ++u) {
      const uint32_t t = first + 4U * quad + u;
      if (hole >> u & 1U) {
        if (hole_rank < most) list[hole_rank].x = t;
        ++hole_rank;
      }
      if (mover >> u & 1U) {
        if (mover_rank < most) list[mover_rank].y = t;
        ++mover_rank;
      }
    }
    const uint32_t all_lanes = __shfl_sync(0xffffffffU, upto, 31);
    holes += all_lanes & 0xffffU;
    movers += all_lanes >> 16U;
  }
  // the last warp of the last block has counted every mover
  if (rank == blocks - 1U && warp == kSelectWarps - 1U && lane == 0U) headers[row] = {n, m, min(movers, most), 0U};
}

// Words of 16 bytes of one record, K and V, and the 2-byte scales of Q4H.
__host__ __device__ __forceinline__ uint32_t record_words(uint32_t encoding, uint32_t hd) {
  return 2U * (encoding == QLLM_KV_F16 ? hd / 8U : hd / 32U + 1U);
}

// Q8 records are on 2-byte boundaries: a warp copies whole records, K and V, in words of four bytes from the target's first
// 4-byte boundary on, and the two bytes before or behind them.  codes[0], [1]: K records of targets and sources.
template <uint32_t HD>
__device__ __forceinline__ void move_q8(uint8_t* const (&codes)[2][kMoveBatch], uint32_t count, size_t to_value) {
  constexpr uint32_t kEach = HD / 64U;         // words of a lane, K and V together
  constexpr uint32_t kMoves = HD <= 128U ? 4U : 2U;
  const uint32_t lane = threadIdx.x & 31U, warp = threadIdx.x >> 5U;
  for (uint32_t j0 = warp * kMoves; j0 < count; j0 += kMoveThreads / 32U * kMoves) {
    uint32_t data[kMoves][kEach];
    uint16_t rest[kMoves];
    uint8_t* to[kMoves];
#pragma unroll
    for (uint32_t m = 0; m < kMoves; ++m) {
      to[m] = nullptr;
      rest[m] = 0U;
      if (j0 + m >= count || !codes[0][j0 + m] || !codes[1][j0 + m]) continue;
      to[m] = codes[0][j0 + m];
      const uint8_t* from = codes[1][j0 + m];
      const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to[m])) & 2U;
      const bool same = ((reinterpret_cast<uintptr_t>(to[m]) ^ reinterpret_cast<uintptr_t>(from)) & 2U) == 0U;
#pragma unroll
      for (uint32_t u = 0; u < kEach; ++u) {
        const uint32_t i = lane + 32U * u;
        const uint8_t* p = from + (i >= HD / 4U ? to_value : 0U) + odd + 4U * (i % (HD / 4U));
        data[m][u] = same ? *reinterpret_cast<const uint32_t*>(p)
                          : *reinterpret_cast<const uint16_t*>(p) | static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + 2)) << 16U;
      }
      if (lane < 2U) rest[m] = *reinterpret_cast<const uint16_t*>(from + (lane ? to_value : 0U) + (odd ? 0U : HD));
    }
#pragma unroll
    for (uint32_t m = 0; m < kMoves; ++m) {
      if (!to[m]) continue;
      const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(to[m])) & 2U;
#pragma unroll
      for (uint32_t u = 0; u < kEach; ++u) {
        const uint32_t i = lane + 32U * u;
        *reinterpret_cast<uint32_t*>(to[m] + (i >= HD / 4U ? to_value : 0U) + odd + 4U * (i % (HD / 4U))) = data[m][u];
      }
      if (lane < 2U) *reinterpret_cast<uint16_t*>(to[m] + (lane ? to_value : 0U) + (odd ? 0U : HD)) = rest[m];
    }
  }
}

// Moves in batches: first a thread per move finds its two pages and moves weight and position, then all threads copy
// words, kAtOnce of them in flight each.  The batches of all rows stand in one line, of which each block takes an equal
// share: rows that move nothing cost no blocks (empty ones took 8 us of 32 for 192 rows).
template <uint32_t ENC, uint32_t HD>
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const __grid_constant__ KvEvictArgs a, const RowHeader* headers,
                                                               const uint2* pairs, uint32_t most) {
  constexpr int kAtOnce = 4;
  __shared__ uint8_t* codes[2][kMoveBatch];   // K codes of target and source, null: no page
  __shared__ uint8_t* scales[2][ENC == QLLM_KV_Q4H ? kMoveBatch : 1];
  __shared__ unsigned long long warp_batches[kMoveThreads / 32U], start_base;
  __shared__ uint32_t start_row;
  const uint32_t kv = a.cache.kv_heads, rows = a.cache.sequences * kv, lane = threadIdx.x & 31U, warp = threadIdx.x >> 5U;
  pdl_wait();
  for (uint32_t s = blockIdx.x * kMoveThreads + threadIdx.x; s < a.cache.sequences; s += gridDim.x * kMoveThreads)
    a.lengths_out[s] = headers[static_cast<size_t>(s) * kv].kept;
  // ---- this block's share of the batches
  const auto batches_of = [&](uint32_t row) { return (headers[row].moves + kMoveBatch - 1U) / kMoveBatch; };
  const uint32_t per_thread = (rows + kMoveThreads - 1U) / kMoveThreads;
  const uint32_t r0 = min(rows, threadIdx.x * per_thread), r1 = min(rows, r0 + per_thread);
  unsigned long long own = 0ULL;
  for (uint32_t r = r0; r < r1; ++r) own += batches_of(r);
  unsigned long long upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long t = __shfl_up_sync(0xffffffffU, upto, o);
    if (lane >= static_cast<uint32_t>(o)) upto += t;
  }
  if (lane == 31U) warp_batches[warp] = upto;
  __syncthreads();
  unsigned long long total = 0ULL, before = upto - own;
#pragma unroll
  for (uint32_t w = 0; w < kMoveThreads / 32U; ++w) {
    if (w < warp) before += warp_batches[w];
    total += warp_batches[w];
  }
  unsigned long long batch = blockIdx.x * total / gridDim.x;
  const unsigned long long end = (blockIdx.x + 1ULL) * total / gridDim.x;
  if (batch == end) return;
  if (before <= batch && batch < before + own) {
    uint32_t r = r0;
    unsigned long long base = before;
    for (;; ++r) {
      const uint32_t n = batches_of(r);
      if (batch < base + n) break;
      base += n;
    }
    start_row = r;
    start_base = base;
  }
  __syncthreads();
  uint32_t row = start_row;
  unsigned long long base = start_base;
  constexpr uint32_t hd = HD;
  const uint32_t pt = a.cache.page_tokens;
  const uint32_t words = record_words(ENC, hd), at_once = kMoveThreads / words;  // moves of a block side by side
  const uint32_t local = threadIdx.x / words, part = threadIdx.x % words;
  const bool value = part >= words / 2U;
  const uint32_t word = value ? part - words / 2U : part;
  const bool is_scale = ENC == QLLM_KV_Q4H && word == hd / 32U;
  // from a record's K codes (scale) to the thread's word
  const size_t to_value = kv_codes_at(a.cache, true, 0U, 0U);
  const size_t delta = (value ? to_value : 0U) + (is_scale ? 0U : 16U * word);
  for (; batch < end; ++batch) {
    uint32_t moves = headers[row].moves;
    while (batch - base >= (moves + kMoveBatch - 1U) / kMoveBatch) {
      base += (moves + kMoveBatch - 1U) / kMoveBatch;
      moves = headers[++row].moves;
    }
    const uint32_t i0 = static_cast<uint32_t>(batch - base) * kMoveBatch;
    const uint32_t count = min(kMoveBatch, moves - i0), s = row / kv, h = row % kv;
    const uint2* list = pairs + static_cast<size_t>(row) * most;
    const size_t at = static_cast<size_t>(row) * a.stride;
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
    if constexpr (ENC == QLLM_KV_Q8) {
      move_q8<HD>(codes, count, to_value);
      continue;
    }
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
        if (is_scale) {
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
        if (is_scale) *reinterpret_cast<uint16_t*>(to[u]) = static_cast<uint16_t>(data[u].x);
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
  const uint32_t slice = ((capacity + cluster - 1U) / cluster + 127U) & ~127U;
  const uint32_t keys_held = min(slice, kMaxKeys);
  if (keys_held > kKeysByDefault) {
    e = cudaFuncSetAttribute(kv_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxKeys * sizeof(uint32_t));
    if (e != cudaSuccess) return check_cuda(e, "kv_evict shared memory opt-in");
  }
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

  const uint64_t batches = static_cast<uint64_t>(rows) * ((most + kMoveBatch - 1U) / kMoveBatch);
  const dim3 grid(static_cast<uint32_t>(max(static_cast<uint64_t>(1U), min(batches, static_cast<uint64_t>(kMoveBlocks) * sms)))), block(kMoveThreads);
  count_launch();
  const auto move = [&](auto kernel) { return launch_pdl(kernel, grid, block, 0, stream, a, headers, pairs, most); };
  const uint32_t hd = a.cache.head_dim;
  switch (a.cache.encoding) {
    case QLLM_KV_F16:
      e = hd == 64U    ? move(kv_move_kernel<QLLM_KV_F16, 64>)
          : hd == 128U ? move(kv_move_kernel<QLLM_KV_F16, 128>)
          : hd == 192U ? move(kv_move_kernel<QLLM_KV_F16, 192>)
                       : move(kv_move_kernel<QLLM_KV_F16, 256>);
      break;
    case QLLM_KV_Q4H:
      e = hd == 64U    ? move(kv_move_kernel<QLLM_KV_Q4H, 64>)
          : hd == 128U ? move(kv_move_kernel<QLLM_KV_Q4H, 128>)
          : hd == 192U ? move(kv_move_kernel<QLLM_KV_Q4H, 192>)
                       : move(kv_move_kernel<QLLM_KV_Q4H, 256>);
      break;
    default:
      e = hd == 64U    ? move(kv_move_kernel<QLLM_KV_Q8, 64>)
          : hd == 128U ? move(kv_move_kernel<QLLM_KV_Q8, 128>)
          : hd == 192U ? move(kv_move_kernel<QLLM_KV_Q8, 192>)
                       : move(kv_move_kernel<QLLM_KV_Q8, 256>);
  }
  return check_cuda(e, "kv_evict move");
}

}  // namespace qllm
