// Attention of one new token per sequence over the paged cache, for a batch of sequences of
// different lengths (qllm_k_decode_attention), and the attention weight that each cached key received.
//
//   z_t = scale * q . K_t,  p_t = exp(z_t) / sum_u exp(z_u),  out = sum_t p_t V_t
//   weights_out_t = weights_in_t + sum over the group's query heads of p_t
//
// First form: one CTA per (query head, sequence), FP32 arithmetic on the CUDA cores, 128 keys at a
// time with the running maximum and sum of the softmax.
#include "kv_batch.cuh"
#include "launch.cuh"

namespace qllm {

namespace {

constexpr uint32_t kThreads = 128;

__device__ __forceinline__ float cache_value(const KvBatch& c, const uint8_t* layer, bool value, uint32_t place,
                                             uint32_t h, uint32_t d, float scale) {
  const uint8_t* codes = layer + kv_codes_at(c, value, place, h);
  if (c.encoding == QLLM_KV_F16) return __half2float(reinterpret_cast<const __half*>(codes)[d]);
  if (c.encoding == QLLM_KV_Q8) return static_cast<float>(static_cast<int8_t>(codes[d])) * scale;
  const int nibble = (codes[d / 2U] >> (4U * (d & 1U))) & 15;
  return static_cast<float>(nibble >= 8 ? nibble - 16 : nibble) * scale;
}
__device__ __forceinline__ float cache_scale(const KvBatch& c, const uint8_t* layer, bool value, uint32_t place, uint32_t h) {
  if (c.encoding == QLLM_KV_F16) return 1.0F;
  return __half2float(*reinterpret_cast<const __half*>(layer + kv_scale_at(c, value, place, h)));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) decode_attention_kernel(DecodeAttentionArgs a, float* scores, float* lse) {
  __shared__ float q[256], z[kThreads], vscale[kThreads], warps[4];
  __shared__ const uint8_t* pages[kThreads];
  const uint32_t head = blockIdx.x, s = blockIdx.y, hd = a.cache.head_dim;
  const uint32_t h = head / (a.q_heads / a.cache.kv_heads);
  const uint32_t n = min(a.lengths[s], kv_capacity(a.cache));
  for (uint32_t d = threadIdx.x; d < hd; d += kThreads)
    q[d] = row_value(static_cast<const T*>(a.query)[s * a.query_stride + static_cast<size_t>(head) * hd + d]);
  float m = -INFINITY, l = 0.0F, acc[2] = {0.0F, 0.0F};
  for (uint32_t t0 = 0; t0 < n; t0 += kThreads) {
    __syncthreads();
    const uint32_t t = t0 + threadIdx.x;
    const uint32_t place = t % a.cache.page_tokens;
    const uint8_t* layer = t < n ? kv_page(a.cache, s, t / a.cache.page_tokens) : nullptr;
    float score = -INFINITY;
    if (layer) {
      const float scale = cache_scale(a.cache, layer, false, place, h);
      float dot = 0.0F;
      for (uint32_t d = 0; d < hd; ++d) dot = fmaf(q[d], cache_value(a.cache, layer, false, place, h, d, scale), dot);
      score = dot * a.scale;
      vscale[threadIdx.x] = cache_scale(a.cache, layer, true, place, h);
    }
    if (scores && t < n) scores[(static_cast<size_t>(s) * a.q_heads + head) * kv_capacity(a.cache) + t] = score;
    pages[threadIdx.x] = layer;
    const float top = warp_max(score);
    if ((threadIdx.x & 31U) == 0U) warps[threadIdx.x >> 5U] = top;
    __syncthreads();
    const float next = fmaxf(m, fmaxf(fmaxf(warps[0], warps[1]), fmaxf(warps[2], warps[3])));
    const float reference = next == -INFINITY ? 0.0F : next;
    const float old = expf(m - reference);
    z[threadIdx.x] = expf(score - reference);
    m = next;
    __syncthreads();
    l *= old;
    acc[0] *= old;
    acc[1] *= old;
    const uint32_t count = min(kThreads, n - t0);
    for (uint32_t j = 0; j < count; ++j) {
      const float p = z[j];
      l += p;
      if (!pages[j]) continue;
#pragma unroll
      for (uint32_t i = 0; i < 2U; ++i) {
        const uint32_t d = threadIdx.x + i * kThreads;
        if (d < hd)
          acc[i] = fmaf(p, cache_value(a.cache, pages[j], true, (t0 + j) % a.cache.page_tokens, h, d, vscale[j]), acc[i]);
      }
    }
  }
  T* out = static_cast<T*>(a.out) + s * a.out_stride + static_cast<size_t>(head) * hd;
  const bool empty = m == -INFINITY;
#pragma unroll
  for (uint32_t i = 0; i < 2U; ++i) {
    const uint32_t d = threadIdx.x + i * kThreads;
    if (d < hd) put_row(out + d, empty ? 0.0F : acc[i] / l);
  }
  if (lse && threadIdx.x == 0U) lse[static_cast<size_t>(s) * a.q_heads + head] = empty ? 0.0F : m + logf(l);
}

__global__ void __launch_bounds__(kThreads) decode_weights_kernel(DecodeAttentionArgs a, const float* scores, const float* lse) {
  const uint32_t h = blockIdx.y, s = blockIdx.z, group = a.q_heads / a.cache.kv_heads;
  const uint32_t n = min(a.lengths[s], kv_capacity(a.cache));
  const uint32_t t = blockIdx.x * kThreads + threadIdx.x;
  if (t >= n) return;
  float sum = 0.0F;
  for (uint32_t g = 0; g < group; ++g) {
    const size_t row = static_cast<size_t>(s) * a.q_heads + h * group + g;
    sum += expf(scores[row * kv_capacity(a.cache) + t] - lse[row]);
  }
  const size_t at = (static_cast<size_t>(s) * a.cache.kv_heads + h) * a.weights_stride + t;
  a.weights_out[at] = (a.weights_in ? a.weights_in[at] : 0.0F) + sum;
}

template <typename T>
int launch(const DecodeAttentionArgs& a, cudaStream_t stream) {
  const size_t heads = static_cast<size_t>(a.cache.sequences) * a.q_heads;
  float* lse = a.weights_out ? static_cast<float*>(a.workspace) : nullptr;
  float* scores = lse ? lse + heads : nullptr;
  decode_attention_kernel<T><<<dim3(a.q_heads, a.cache.sequences), kThreads, 0, stream>>>(a, scores, lse);
  count_launch();
  int rc = check_launch("decode_attention");
  if (rc || !lse) return rc;
  const uint32_t blocks = (kv_capacity(a.cache) + kThreads - 1U) / kThreads;
  decode_weights_kernel<<<dim3(blocks, a.cache.kv_heads, a.cache.sequences), kThreads, 0, stream>>>(a, scores, lse);
  count_launch();
  return check_launch("decode_attention weights");
}

}  // namespace

size_t decode_attention_workspace_bytes(const KvBatch& c, uint32_t q_heads, bool weights) {
  return weights ? static_cast<size_t>(c.sequences) * q_heads * (static_cast<size_t>(kv_capacity(c)) + 1U) * sizeof(float) : 16U;
}

int launch_decode_attention(const DecodeAttentionArgs& a, cudaStream_t stream) {
  if (a.row_type == QLLM_ROW_F32) return launch<float>(a, stream);
  if (a.row_type == QLLM_ROW_BF16) return launch<__nv_bfloat16>(a, stream);
  return launch<__half>(a, stream);
}

}  // namespace qllm
