// Per-head RMS norm of queries and keys, rotation by position and the K/V records, for rows of many
// sequences in one launch (qllm_k_qk_norm_rope_store).
//
//   n_d = x_d * w_d / sqrt(mean_d x_d^2 + eps)                      over the head's D values
//   y_i = n_i cos a_i - n_{i+R/2} sin a_i,  y_{i+R/2} = n_{i+R/2} cos a_i + n_i sin a_i,  i < R/2
//   a_i = position * inv_freq[i];  y_d = n_d for d >= R
//
// Everything between the load of a value and its one rounding to the row's type (or to the record)
// is FP32.  The angle is reduced in FP64: position * inv_freq as an FP32 product is off by up to
// 2^-24 of an angle of thousands of turns, i.e. by whole tenths of a turn at position 10^6.
//
// HBM-bound: a row is read once and its results written once.  A lane owns the eight values at i and
// the eight at i + R/2 (the pair that a rotation mixes), so a head of 128 is eight lanes with two
// 16-byte loads each, a warp takes four heads at a time, no value crosses lanes except in the sum of
// squares (and the maximum of a quantised record), and nothing but cos and sin is in shared memory.
#include "kv_batch.cuh"
#include "launch.cuh"

namespace qllm {

namespace {

constexpr uint32_t kThreads = 256;

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

// grid (rows, blocks of heads)
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads)
norm_rope_store_kernel(NormRopeStoreArgs a, uint32_t heads_per_block) {
  constexpr int kActive = HD / 16;                        // lanes that hold a head
  constexpr int kLanes = kActive == 12 ? 16 : kActive;    // lanes set aside for it
  constexpr uint32_t kHeadsPerWarp = 32 / kLanes;
  __shared__ float2 turn[HD / 2];                         // cos, sin
  const uint32_t row = blockIdx.x;
  const uint32_t slot = a.row_slot ? a.row_slot[row] : 0U;
  if (slot == kPaddingSlot) return;
  const uint32_t position = a.positions[row];
  for (uint32_t i = threadIdx.x; i < a.rotary_dim / 2U; i += kThreads) {
    double t = static_cast<double>(position) * static_cast<double>(a.inv_freq[i]) * 0.15915494309189533577;
    t -= rint(t);  // turns, in [-1/2, 1/2]
    float s, c;
    sincospif(2.0F * static_cast<float>(t), &s, &c);
    turn[i] = make_float2(c, s);
  }
  const uint32_t sequence = a.row_sequence ? a.row_sequence[row] : row;
  uint8_t* layer = nullptr;
  if (a.row_slot && sequence < a.cache.sequences && slot < kv_capacity(a.cache))
    layer = kv_page(a.cache, sequence, slot / a.cache.page_tokens);
  const uint32_t place = slot % a.cache.page_tokens;
  __syncthreads();

  const uint32_t kv = a.cache.kv_heads;
  const uint32_t first = blockIdx.y * heads_per_block;
  const uint32_t all = a.q_heads + (a.row_slot ? 2U : 1U) * kv;
  const uint32_t last = min(all, first + heads_per_block);
  const uint32_t lane = threadIdx.x & 31U, warp = threadIdx.x >> 5U;
  const uint32_t l = lane % kLanes;
  const bool holds = l < kActive;
  // chunks of eight values: the pair (l, l + R/16) inside the rotation, two neighbours outside
  const uint32_t turned = a.rotary_dim / 16U;
  const bool rotates = l < turned;
  const uint32_t c0 = rotates ? l : a.rotary_dim / 8U + 2U * (l - turned);
  const uint32_t c1 = rotates ? l + turned : c0 + 1U;
  const T* x = static_cast<const T*>(a.qkv) + static_cast<size_t>(row) * a.qkv_stride;

  for (uint32_t base = first + warp * kHeadsPerWarp; base < last; base += (kThreads / 32U) * kHeadsPerWarp) {
    const uint32_t head = base + lane / kLanes;
    const bool live = holds && head < last;
    float v0[8] = {}, v1[8] = {};
    if (live) {
      load8(x + static_cast<size_t>(head) * HD + 8U * c0, v0);
      load8(x + static_cast<size_t>(head) * HD + 8U * c1, v1);
    }
    const bool is_value = head >= a.q_heads + kv;
    float sum = 0.0F;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(v0[i], v0[i], fmaf(v1[i], v1[i], sum));
    sum = head_sum<kLanes>(sum);
    if (live && !is_value) {
      const float* w = head < a.q_heads ? a.q_norm : a.k_norm;
      const float r = 1.0F / sqrtf(sum / static_cast<float>(HD) + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v0[i] = v0[i] * r * w[8U * c0 + i];
        v1[i] = v1[i] * r * w[8U * c1 + i];
      }
      if (rotates) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 t = turn[8U * c0 + i];
          const float low = v0[i], high = v1[i];
          v0[i] = fmaf(low, t.x, -high * t.y);
          v1[i] = fmaf(high, t.x, low * t.y);
        }
      }
    }
    float scale = 0.0F;
    __half stored = __float2half_rn(0.0F);
    if (a.row_slot && a.cache.encoding != QLLM_KV_F16) {
      float amax = 0.0F;
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fmaxf(fabsf(v0[i]), fabsf(v1[i])));
      scale = record_scale(head_max<kLanes>(amax), a.cache.encoding == QLLM_KV_Q4H ? 7.0F : 127.0F, &stored);
    }
    if (!live) continue;
    if (head < a.q_heads) {
      T* q = static_cast<T*>(a.query) + static_cast<size_t>(row) * a.query_stride + static_cast<size_t>(head) * HD;
      store8(q + 8U * c0, v0);
      store8(q + 8U * c1, v1);
      continue;
    }
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

template <typename T, int HD>
int launch(const NormRopeStoreArgs& a, cudaStream_t stream) {
  const uint32_t heads = a.q_heads + (a.row_slot ? 2U : 1U) * a.cache.kv_heads;
  norm_rope_store_kernel<T, HD><<<dim3(a.rows), kThreads, 0, stream>>>(a, heads);
  count_launch();
  return check_launch("qk_norm_rope_store");
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
