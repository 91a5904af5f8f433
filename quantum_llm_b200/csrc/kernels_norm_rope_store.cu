// Per-head RMS norm of queries and keys, rotation by position and the K/V records, for rows of many
// sequences in one launch (qllm_k_qk_norm_rope_store).
//
//   n_d = x_d * w_d / sqrt(mean_d x_d^2 + eps)                      over the head's D values (without weights: n = x)
//   y_i = n_i cos a_i - n_{i+R/2} sin a_i,  y_{i+R/2} = n_{i+R/2} cos a_i + n_i sin a_i,  i < R/2
//   a_i = position * inv_freq[i];  y_d = n_d for d >= R
//
// Everything between the load of a value and its one rounding to the row's type (or to the record)
// is FP32.  The angle is reduced in FP64: position * inv_freq as an FP32 product is off by up to
// 2^-24 of the angle, i.e. by a hundredth of a turn at position 10^6.
//
// HBM-bound: a row is read once and its results written once.  A lane owns the eight values at i and
// the eight at i + R/2 (the pair that a rotation mixes), so a head of 128 is eight lanes with two
// 16-byte loads each, a warp takes four heads at a time and no value crosses lanes except in the sum of
// squares (and the maximum of a quantised record).  A warp takes a whole row, or, where rows are few, some heads
// of one: its lanes share the work of the cosines and sines and hand them round by shuffles, so that
// warps need no barrier, and the values of the next passes are copied into shared memory (each lane its own)
// while these are worked on.
//
// Measured on one B200 (copy 6554 GB/s): 8192 rows of 40 query and 8 kv heads of 128, BF16: 42 us for 235 MB, 0.85 of the copy
// rate (2048 rows: 14.7 us, 0.61; with Q8 or Q4H records 52 us; FP32 rows 109 us, 0.61); 517 FP32 rows of 12 and 2 heads of 256: 8.5 us for 16.8 MB, the start of a launch and one chain of loads; 64 rows and one row:
// 4.1 and 3.6 us, a launch.
#include "kv_batch.cuh"
#include "launch.cuh"

namespace qllm {

namespace {

constexpr uint32_t kThreads = 256;
// Warps of a launch, for rows of 40 + 16 heads of 128 with 1024 / 2048 / 4096 of them: 512 rows 8.2 / 6.9 / 8.0 us, 1024 rows 11.3 / 9.3 / 10.8;
// 1024 rows of 16 + 32 heads of 64: 7.5 / 6.2 / 7.1; from 2048 rows on, and for FP32 rows of 256, the same within 2 %.
constexpr uint32_t kWarpsWanted = 2048;

template <int kLanes>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffU, v, o);
  return v;
}
template <int kLanes>
__device__ __forceinline__ float head_max(float v) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffU, v, o));
  return v;
}

// Scale of a quantised record: the largest magnitude over the largest code, as F16 (never 0, never
// infinite; a NaN value does not count and becomes code 0).
__device__ __forceinline__ float record_scale(float amax, float top, __half* stored) {
  *stored = __float2half_rn(fminf(fmaxf(amax / top, 0x1p-24F), 65504.0F));
  return __half2float(*stored);
}
__device__ __forceinline__ int code_of(float v, float scale, int top) {
  return max(-top, min(top, __float2int_rn(v / scale)));
}

// Eight consecutive values of a record starting at dimension 8 * chunk.
__device__ __forceinline__ void store_record8(const KvBatch& c, uint8_t* codes, uint32_t chunk, const float (&v)[8],
                                              float scale) {
  if (c.encoding == QLLM_KV_F16) {
    store8(reinterpret_cast<__half*>(codes) + 8U * chunk, v);
  } else if (c.encoding == QLLM_KV_Q4H) {
    uint32_t w = 0U;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (static_cast<uint32_t>(code_of(v[i], scale, 7)) & 15U) << (4 * i);
    reinterpret_cast<uint32_t*>(codes)[chunk] = w;
  } else {  // Q8 records are on 2-byte boundaries
    uint16_t* dst = reinterpret_cast<uint16_t*>(codes + 8U * chunk);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      dst[i] = static_cast<uint16_t>((static_cast<uint32_t>(code_of(v[2 * i], scale, 127)) & 0xffU) |
                                     ((static_cast<uint32_t>(code_of(v[2 * i + 1], scale, 127)) & 0xffU) << 8U));
  }
}

__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}

template <typename T>
__host__ __device__ constexpr uint32_t stages() {
  return sizeof(T) == 2U ? 4U : 2U;  // 32 KiB of a block, of which four share a multiprocessor (three for FP32: no faster)
}

// One warp per task: `passes` times kHeadsPerWarp heads of one row.
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 4)
norm_rope_store_kernel(const __grid_constant__ NormRopeStoreArgs a, uint32_t tasks_per_row, uint32_t passes) {
  constexpr uint32_t kActive = HD / 16;                        // lanes that hold a head
  constexpr uint32_t kLanes = kActive == 12U ? 16U : kActive;  // lanes set aside for it
  constexpr uint32_t kHeadsPerWarp = 32U / kLanes;
  constexpr uint32_t kTurns = kLanes / 4U;                     // cosines a lane works out
  constexpr uint32_t kStages = stages<T>();                    // passes in flight
  constexpr uint32_t kWords = sizeof(T) / 2U;                  // 16-byte words of eight values
  __shared__ alignas(16) float norm[2][HD];
  extern __shared__ uint4 ring_memory[];                       // a lane's values of the passes to come; nobody else reads them
  uint4 (&ring)[kStages][2U * kWords][kThreads] = *reinterpret_cast<uint4 (*)[kStages][2U * kWords][kThreads]>(ring_memory);
  for (uint32_t i = threadIdx.x; i < 2U * HD; i += kThreads) norm[i / HD][i % HD] = a.q_norm ? (i < HD ? a.q_norm : a.k_norm)[i % HD] : 1.0F;
  __syncthreads();
  const uint64_t task = static_cast<uint64_t>(blockIdx.x) * (kThreads / 32U) + (threadIdx.x >> 5U);
  const uint32_t row = static_cast<uint32_t>(task / tasks_per_row);
  if (row >= a.rows) return;
  const uint32_t lane = threadIdx.x & 31U, l = lane % kLanes, which = lane / kLanes;
  const uint32_t kv = a.cache.kv_heads, all = a.q_heads + (a.row_slot ? 2U : 1U) * kv;
  const uint32_t first = static_cast<uint32_t>(task % tasks_per_row) * passes * kHeadsPerWarp;
  const uint32_t last = min(all, first + passes * kHeadsPerWarp);
  // chunks of eight values: the pair (l, l + R/16) inside the rotation, two neighbours outside
  const uint32_t turned = a.rotary_dim / 16U;
  const bool rotates = l < turned;
  const uint32_t c0 = rotates ? l : a.rotary_dim / 8U + 2U * (l - turned);
  const uint32_t c1 = rotates ? l + turned : c0 + 1U;
  const T* x = static_cast<const T*>(a.qkv) + static_cast<size_t>(row) * a.qkv_stride;
  const auto fetch = [&](uint32_t head, uint32_t stage) {
    if (l < kActive && head < last) {
#pragma unroll
      for (uint32_t i = 0; i < kWords; ++i) {
        copy16(&ring[stage][i][threadIdx.x], x + static_cast<size_t>(head) * HD + 8U * c0 + i * 16U / sizeof(T));
        copy16(&ring[stage][kWords + i][threadIdx.x], x + static_cast<size_t>(head) * HD + 8U * c1 + i * 16U / sizeof(T));
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (uint32_t i = 0; i < kStages - 1U; ++i) fetch(first + i * kHeadsPerWarp + which, i);

  const uint32_t slot = a.row_slot ? a.row_slot[row] : 0U;
  if (slot == kPaddingSlot) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");  // its copies are not to outlive the block
    return;
  }
  const uint32_t position = a.positions[row];
  const uint32_t sequence = a.row_sequence ? a.row_sequence[row] : row;
  // cos and sin of the lane's pairs 8 l .. 8 l + 7: the lanes of the kHeadsPerWarp heads work out kTurns of them each
  float cosine[8], sine[8];
  {
    float c[kTurns], s[kTurns];
#pragma unroll
    for (uint32_t i = 0; i < kTurns; ++i) {
      double t = 0.0;
      if (rotates) t = static_cast<double>(position) * static_cast<double>(a.inv_freq[8U * l + which * kTurns + i]) * 0.15915494309189533577;
      t -= rint(t);  // turns, in [-1/2, 1/2]
      sincospif(2.0F * static_cast<float>(t), &s[i], &c[i]);
    }
#pragma unroll
    for (uint32_t e = 0; e < 8U; ++e) {
      cosine[e] = __shfl_sync(0xffffffffU, c[e % kTurns], e / kTurns * kLanes + l);
      sine[e] = __shfl_sync(0xffffffffU, s[e % kTurns], e / kTurns * kLanes + l);
    }
  }
  uint8_t* layer = nullptr;
  uint32_t place = 0U;
  if (a.row_slot && sequence < a.cache.sequences && slot < kv_capacity(a.cache)) {
    layer = kv_page(a.cache, sequence, slot / a.cache.page_tokens);
    place = slot % a.cache.page_tokens;
  }

  for (uint32_t base = first; base < last; base += kStages * kHeadsPerWarp) {
#pragma unroll
    for (uint32_t stage = 0; stage < kStages; ++stage) {
      const uint32_t head = base + stage * kHeadsPerWarp + which;
      if (head - which >= last) break;
      const bool live = l < kActive && head < last;
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2U) : "memory");
      float v0[8], v1[8];
      {
        uint4 raw[2U * kWords];
#pragma unroll
        for (uint32_t i = 0; i < 2U * kWords; ++i) raw[i] = live ? ring[stage][i][threadIdx.x] : make_uint4(0U, 0U, 0U, 0U);
        load8(reinterpret_cast<const T*>(raw), v0);
        load8(reinterpret_cast<const T*>(raw + kWords), v1);
      }
      fetch(head + (kStages - 1U) * kHeadsPerWarp, (stage + kStages - 1U) % kStages);
      const bool is_value = head >= a.q_heads + kv;
      float sum = 0.0F;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(v0[i], v0[i], fmaf(v1[i], v1[i], sum));
      sum = head_sum<kLanes>(sum);
      if (live && !is_value) {
        const float* w = norm[head < a.q_heads ? 0 : 1];
        const float r = a.q_norm ? rsqrtf(fmaf(sum, 1.0F / HD, a.eps)) : 1.0F;
        float w0[8], w1[8];
        load8(w + 8U * c0, w0);
        load8(w + 8U * c1, w1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v0[i] *= r * w0[i];
          v1[i] *= r * w1[i];
        }
        if (rotates) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float low = v0[i], high = v1[i];
            v0[i] = fmaf(low, cosine[i], -(high * sine[i]));
            v1[i] = fmaf(high, cosine[i], low * sine[i]);
          }
        }
      }
      if (live && head < a.q_heads) {
        T* q = static_cast<T*>(a.query) + static_cast<size_t>(row) * a.query_stride + static_cast<size_t>(head) * HD;
        store8(q + 8U * c0, v0);
        store8(q + 8U * c1, v1);
      }
      if (base + (stage + 1U) * kHeadsPerWarp <= a.q_heads) continue;
      // ---- keys and values (whole warps from here on: the maximum of a record goes over lanes)
      float scale = 0.0F;
      __half stored = __float2half_rn(0.0F);
      if (a.row_slot && a.cache.encoding != QLLM_KV_F16) {
        float amax = 0.0F;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fmaxf(fabsf(v0[i]), fabsf(v1[i])));
        scale = record_scale(head_max<kLanes>(amax), a.cache.encoding == QLLM_KV_Q4H ? 7.0F : 127.0F, &stored);
      }
      if (!live || head < a.q_heads) continue;
      const uint32_t h = head - a.q_heads - (is_value ? kv : 0U);
      if (!is_value && a.key) {
        T* k = static_cast<T*>(a.key) + static_cast<size_t>(row) * a.key_stride + static_cast<size_t>(h) * HD;
        store8(k + 8U * c0, v0);
        store8(k + 8U * c1, v1);
      }
      if (!layer) continue;
      uint8_t* codes = layer + kv_codes_at(a.cache, is_value, place, h);
      store_record8(a.cache, codes, c0, v0, scale);
      store_record8(a.cache, codes, c1, v1, scale);
      if (l == 0U) {
        if (a.cache.encoding != QLLM_KV_F16)
          *reinterpret_cast<__half*>(layer + kv_scale_at(a.cache, is_value, place, h)) = stored;
        if (!is_value && a.slot_positions)
          a.slot_positions[(static_cast<size_t>(sequence) * kv + h) * a.slot_stride + slot] = position;
      }
    }
  }
}

template <typename T, int HD>
int launch(const NormRopeStoreArgs& a, cudaStream_t stream) {
  constexpr uint32_t kHeadsPerWarp = HD == 64 ? 8U : HD == 128 ? 4U : 2U;
  const uint32_t heads = a.q_heads + (a.row_slot ? 2U : 1U) * a.cache.kv_heads;
  const uint32_t all = (heads + kHeadsPerWarp - 1U) / kHeadsPerWarp;
  // as many passes to a warp as leave kWarpsWanted of them
  const uint32_t passes = static_cast<uint32_t>(max(static_cast<uint64_t>(1U), min(static_cast<uint64_t>(all), static_cast<uint64_t>(all) * a.rows / kWarpsWanted)));
  const uint32_t tasks = (all + passes - 1U) / passes;
  const uint64_t blocks = (static_cast<uint64_t>(tasks) * a.rows + kThreads / 32U - 1U) / (kThreads / 32U);
  if (blocks > 0x7FFFFFFFULL) return fail(QLLM_INVALID_ARGUMENT, "QK norm / RoPE / KV store: too many rows");
  constexpr uint32_t kShared = stages<T>() * sizeof(T) * kThreads * 16U;
  count_launch();
  return check_cuda(launch_ordered(norm_rope_store_kernel<T, HD>, dim3(static_cast<uint32_t>(blocks)), dim3(kThreads), kShared, stream, a, tasks, passes),
                    "qk_norm_rope_store");
}

template <typename T>
int dispatch(const NormRopeStoreArgs& a, cudaStream_t stream) {
  switch (a.cache.head_dim) {
    case 64: return launch<T, 64>(a, stream);
    case 128: return launch<T, 128>(a, stream);
    case 192: return launch<T, 192>(a, stream);
    default: return launch<T, 256>(a, stream);
  }
}

}  // namespace

int launch_norm_rope_store(const NormRopeStoreArgs& a, cudaStream_t stream) {
  if (a.row_type == QLLM_ROW_F32) return dispatch<float>(a, stream);
  if (a.row_type == QLLM_ROW_BF16) return dispatch<__nv_bfloat16>(a, stream);
  return dispatch<__half>(a, stream);
}

}  // namespace qllm
