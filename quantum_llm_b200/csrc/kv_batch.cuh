// What the operators for batches of sequences share: the paged cache of one layer as several
// sequences see it (qllm_kv_batch), rows of FP32 / BF16 / F16 values, and the record layouts.
//
// Page layout per layer, the same bytes as the single-sequence kernels read and write:
//   F16: [K pt*kv*hd f16][V ...], token-major
//   Q4H: [K codes kv*pt*hd/2][K scales f16 kv*pt][V codes][V scales], record = kv_head*pt + slot%pt
//   Q8 : [K records pt*kv*(hd+2)][V records], record = (slot%pt)*kv + kv_head, int8[hd] + f16 scale
#pragma once

#include "common.cuh"

namespace qllm {

using KvBatch = qllm_kv_batch;

constexpr uint32_t kPaddingSlot = 0xFFFFFFFFU;

__host__ __device__ __forceinline__ uint32_t kv_capacity(const KvBatch& c) { return c.pages_per_sequence * c.page_tokens; }

#ifdef __CUDACC__
// The layer's part of page `page` of a sequence; null where the table has no usable page (null, or
// not on a 16-byte boundary): the callers store nothing there and read nothing.
__device__ __forceinline__ uint8_t* kv_page(const KvBatch& c, uint32_t sequence, uint32_t page) {
  uint8_t* p = c.page_tables[static_cast<size_t>(sequence) * c.pages_per_sequence + page];
  return (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15U)) ? nullptr : p + c.layer_offset;
}

// Byte offset, inside the layer's part of a page, of the codes (values) of one record, and of its scale.
__device__ __forceinline__ size_t kv_codes_at(const KvBatch& c, bool value, uint32_t place, uint32_t kv_head) {
  const size_t records = static_cast<size_t>(c.page_tokens) * c.kv_heads;
  const size_t token_major = static_cast<size_t>(place) * c.kv_heads + kv_head;
  if (c.encoding == QLLM_KV_F16) return (value ? records + token_major : token_major) * c.head_dim * 2U;
  if (c.encoding == QLLM_KV_Q8) return (value ? records + token_major : token_major) * (c.head_dim + 2U);
  return (value ? records * (c.head_dim / 2U + 2U) : 0U) +
         (static_cast<size_t>(kv_head) * c.page_tokens + place) * (c.head_dim / 2U);
}
__device__ __forceinline__ size_t kv_scale_at(const KvBatch& c, bool value, uint32_t place, uint32_t kv_head) {
  if (c.encoding == QLLM_KV_Q8) return kv_codes_at(c, value, place, kv_head) + c.head_dim;
  const size_t records = static_cast<size_t>(c.page_tokens) * c.kv_heads;
  return (value ? records * (c.head_dim / 2U + 2U) : 0U) + records * (c.head_dim / 2U) +
         (static_cast<size_t>(kv_head) * c.page_tokens + place) * 2U;
}

// Eight consecutive row values (16-byte aligned; FP32: two 16-byte words) as FP32, and back.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16U);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000U);
  }
}
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  __half2 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
}
__device__ __forceinline__ float row_value(float v) { return v; }
__device__ __forceinline__ float row_value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float row_value(__half v) { return __half2float(v); }
__device__ __forceinline__ void put_row(float* p, float v) { *p = v; }
__device__ __forceinline__ void put_row(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put_row(__half* p, float v) { *p = __float2half_rn(v); }
#endif

// ---- launch interface (kernels_norm_rope_store.cu, kernels_decode_attention.cu, kernels_kv_evict.cu);
// the arguments have been checked by the C entries in c_api_batch.cu.
struct NormRopeStoreArgs {
  KvBatch cache;
  uint32_t row_type;
  const void* qkv;           // [rows, (q + 2 kv) * head_dim], rows qkv_stride elements apart
  size_t qkv_stride;
  uint32_t rows, q_heads, rotary_dim;
  const float* q_norm;       // [head_dim]; both null: no norm
  const float* k_norm;
  float eps;
  const float* inv_freq;     // [rotary_dim / 2]
  const uint32_t* positions; // [rows]
  const uint32_t* row_sequence;  // [rows], null: row r belongs to sequence r
  const uint32_t* row_slot;      // [rows], null: no records
  void* query;
  size_t query_stride;
  void* key;                 // null: not wanted
  size_t key_stride;
  uint32_t* slot_positions;  // [sequences, kv_heads, slot_stride], null: not wanted
  size_t slot_stride;
};
int launch_norm_rope_store(const NormRopeStoreArgs& a, cudaStream_t stream);

struct DecodeAttentionArgs {
  KvBatch cache;
  uint32_t row_type;
  const void* query;         // [sequences, q_heads * head_dim], query_stride elements apart
  size_t query_stride;
  const uint32_t* lengths;   // [sequences]
  uint32_t q_heads;
  float scale;
  const float* weights_in;   // [sequences, kv_heads, weights_stride], null: start from zero
  float* weights_out;        // null: not wanted
  size_t weights_stride;
  void* out;                 // [sequences, q_heads * head_dim]
  size_t out_stride;
  void* workspace;
};
size_t decode_attention_workspace_bytes(const KvBatch& cache, uint32_t q_heads, bool weights);
int launch_decode_attention(const DecodeAttentionArgs& a, cudaStream_t stream);

struct KvEvictArgs {
  KvBatch cache;
  const uint32_t* lengths_in;  // [sequences]
  uint32_t* lengths_out;
  const uint32_t* next_positions;  // [sequences]
  uint32_t budget, recent, sinks;
  const float* weights_in;     // [sequences, kv_heads, stride]
  float* weights_out;
  const uint32_t* positions_in;
  uint32_t* positions_out;
  size_t stride;
  void* workspace;
};
size_t kv_evict_workspace_bytes(const KvBatch& cache, uint32_t budget);
int launch_kv_evict(const KvEvictArgs& a, cudaStream_t stream);

}  // namespace qllm
