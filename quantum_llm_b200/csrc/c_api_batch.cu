// extern "C" forms of the operators for batches of sequences (include/qllm_b200.h): every argument
// that the host can see is checked here, before any CUDA call.
#include <cmath>
#include <initializer_list>
#include <string>

#include "kernels.h"
#include "kv_batch.cuh"

using namespace qllm;

namespace {

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1U)) == 0U; }

// Whether [p, p + bytes) and [q, q + bytes_q) share memory.
bool overlap(const void* p, size_t bytes, const void* q, size_t bytes_q) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return a < b + bytes_q && b < a + bytes;
}

// Lists and arrays of 32-bit elements, null where one is not wanted: the kernels read and write whole words.
template <typename... P>
int check_words(const char* who, const P*... p) {
  if ((aligned(p, 4U) && ...)) return 0;
  return fail(QLLM_INVALID_ARGUMENT, std::string(who) + " needs lists and arrays on 4-byte boundaries");
}

size_t row_bytes(uint32_t type) { return type == QLLM_ROW_F32 ? 4U : 2U; }

// Whether `rows` rows `stride` elements apart can be addressed at all.
bool extent_ok(size_t rows, size_t stride) { return stride <= (static_cast<size_t>(1) << 56U) / rows; }

// `count` rows of `width` elements of `size` bytes, `stride` elements apart; the strides have passed extent_ok.
struct Rows {
  const void* p;
  size_t count, stride, width, size;
  size_t bytes() const { return ((count - 1U) * stride + width) * size; }
};
// Whether two sets of rows share memory.  Rows of one stride may be columns of one buffer; of different strides the space
// between the rows counts as theirs.
bool overlap(const Rows& a, const Rows& b) {
  if (!overlap(a.p, a.bytes(), b.p, b.bytes())) return false;
  const size_t period = a.stride * a.size;
  if (period != b.stride * b.size) return true;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  const size_t after = y >= x ? (y - x) % period : (period - (x - y) % period) % period;  // from a row of a to the next of b
  return after < a.width * a.size || after + b.width * b.size > period;
}

// Geometry of the cache; 0 or the refusal.
int check_cache(const qllm_kv_batch* c, const char* who) {
  if (!c || !c->sequences || !c->kv_heads) return fail(QLLM_INVALID_ARGUMENT, std::string("invalid ") + who + " batch");
  if (c->sequences > 65535U || c->kv_heads > 4096U)
    return fail(QLLM_INVALID_ARGUMENT, std::string(who) + " takes at most 65535 sequences and 4096 kv heads");
  if (c->head_dim != 64U && c->head_dim != 128U && c->head_dim != 192U && c->head_dim != 256U)
    return fail(QLLM_INVALID_ARGUMENT, std::string(who) + " needs head_dim 64, 128, 192 or 256");
  return 0;
}
// Its pages, but for the table of them.
int check_page_geometry(const qllm_kv_batch* c, const char* who) {
  if (!c->pages_per_sequence || c->encoding > QLLM_KV_Q8) return fail(QLLM_INVALID_ARGUMENT, std::string("invalid ") + who + " cache");
  if (!c->page_tokens || c->page_tokens % 16U || c->layer_offset % 16U)
    return fail(QLLM_INVALID_ARGUMENT, std::string(who) + " needs page_tokens and layer_offset in multiples of 16");
  if (static_cast<uint64_t>(c->pages_per_sequence) * c->page_tokens >= 0x80000000ULL)
    return fail(QLLM_INVALID_ARGUMENT, std::string(who) + " takes fewer than 2^31 slots per sequence");
  if (kv_layer_bytes(c->encoding, 1U, c->kv_heads, c->head_dim) * c->page_tokens >= 0x100000000ULL)
    return fail(QLLM_INVALID_ARGUMENT, std::string(who) + " takes pages that hold less than 4 GiB of a layer");
  return 0;
}

int check_pages(const qllm_kv_batch* c, const char* who) {
  if (!c->page_tables || !aligned(c->page_tables, 8U)) return fail(QLLM_INVALID_ARGUMENT, std::string("invalid ") + who + " cache");
  return check_page_geometry(c, who);
}

// The query heads of an attention batch.
int check_query_heads(const qllm_kv_batch* c, uint32_t q_heads) {
  if (!q_heads || q_heads > 65536U || q_heads % c->kv_heads) return fail(QLLM_INVALID_ARGUMENT, "invalid decode attention batch");
  if (static_cast<uint64_t>(c->sequences) * q_heads > (1U << 28U))
    return fail(QLLM_INVALID_ARGUMENT, "decode attention takes at most 2^28 query heads over all sequences");
  return 0;
}

// Rows that are read or written in 16-byte words.
bool rows_ok(const void* p, size_t rows, size_t stride, uint32_t type, size_t width) {
  return p && aligned(p, 16U) && stride >= width && stride * row_bytes(type) % 16U == 0U && extent_ok(rows, stride);
}

// The call's memory has to be the current device's: a host pointer, or another device's memory, would fault in the kernel.
// The rows or page tables stand for all of a call's memory, and one list for its lists, which are what a host has at hand (0.15 us a
// pointer; all pointers of a call would be 0.9 us of some 5).  Lists may lie in pinned host memory, which the device reads as it is.
int check_device(const char* what, std::initializer_list<const void*> memory, const void* list) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  bool there = true;
  const auto check = [&](const void* p, bool pinned) {
    if (e != cudaSuccess || !there || !p) return;
    cudaPointerAttributes attributes{};
    e = cudaPointerGetAttributes(&attributes, p);
    there = (attributes.type == cudaMemoryTypeDevice && attributes.device == device) || attributes.type == cudaMemoryTypeManaged ||
            (pinned && attributes.type == cudaMemoryTypeHost);
  };
  for (const void* p : memory) check(p, false);
  check(list, true);
  if (e != cudaSuccess) {
    cudaGetLastError();  // reported here, not by the next call
    return check_cuda(e, what);
  }
  return there ? 0 : fail(QLLM_INVALID_ARGUMENT, std::string(what) + ": the call's memory is not the current device's");
}

}  // namespace

extern "C" {

int qllm_k_qk_norm_rope_store(const qllm_kv_batch* cache, uint32_t row_type, const void* qkv, size_t qkv_stride,
                              uint32_t rows, uint32_t q_heads, uint32_t rotary_dim, const float* q_norm,
                              const float* k_norm, float eps, const float* inv_freq, const uint32_t* positions,
                              const uint32_t* row_sequence, const uint32_t* row_slot, void* query, size_t query_stride,
                              void* key, size_t key_stride, uint32_t* slot_positions, size_t slot_stride,
                              void* stream) {
  const char* who = "QK norm / RoPE / KV store";
  int rc = check_cache(cache, who);
  if (rc) return rc;
  if (row_slot && (rc = check_pages(cache, who))) return rc;
  if (!rows || !q_heads || q_heads > 65536U || row_type > QLLM_ROW_F16 || !q_norm != !k_norm || !positions ||
      !(eps >= 0.0F) || std::isinf(eps))
    return fail(QLLM_INVALID_ARGUMENT, "invalid QK norm / RoPE / KV store batch");
  if ((rc = check_words(who, q_norm, k_norm, inv_freq, positions, row_sequence, row_slot, slot_positions))) return rc;
  if (rotary_dim > cache->head_dim || rotary_dim % 16U || (rotary_dim && !inv_freq))
    return fail(QLLM_INVALID_ARGUMENT, "QK norm / RoPE / KV store needs a rotary_dim that is a multiple of 16 and at most head_dim");
  if (row_slot && !row_sequence && rows > cache->sequences)
    return fail(QLLM_INVALID_ARGUMENT, "QK norm / RoPE / KV store: without row_sequence there is at most one row per sequence");
  const size_t q_width = static_cast<size_t>(q_heads) * cache->head_dim, kv_width = static_cast<size_t>(cache->kv_heads) * cache->head_dim;
  const size_t e = row_bytes(row_type);
  if (!rows_ok(qkv, rows, qkv_stride, row_type, q_width + 2U * kv_width) || !rows_ok(query, rows, query_stride, row_type, q_width) ||
      (key && !rows_ok(key, rows, key_stride, row_type, kv_width)))
    return fail(QLLM_INVALID_ARGUMENT,
                "QK norm / RoPE / KV store needs rows on 16-byte boundaries, strides that hold a row and are multiples of 16 bytes");
  if (slot_positions && (!row_slot || slot_stride < kv_capacity(*cache) ||
                         !extent_ok(static_cast<size_t>(cache->sequences) * cache->kv_heads, slot_stride)))
    return fail(QLLM_INVALID_ARGUMENT, "QK norm / RoPE / KV store: slot_positions needs row_slot and a stride that holds every slot");
  // in place is every row's own head over itself; any other sharing would be overwritten before it is read
  const Rows in{qkv, rows, qkv_stride, q_width + 2U * kv_width, e}, q_out{query, rows, query_stride, q_width, e},
      k_out{key, rows, key_stride, kv_width, e};
  const bool query_in_place = query == qkv && query_stride == qkv_stride;
  const bool key_in_place = key == static_cast<const uint8_t*>(qkv) + q_width * e && key_stride == qkv_stride;
  if ((!query_in_place && overlap(q_out, in)) || (key && !key_in_place && overlap(k_out, in)) || (key && overlap(k_out, q_out)))
    return fail(QLLM_INVALID_ARGUMENT, "QK norm / RoPE / KV store: rows overlap and are not in place");
  if ((rc = check_device(who, {qkv, row_slot ? cache->page_tables : nullptr}, positions))) return rc;
  NormRopeStoreArgs a{*cache, row_type, qkv, qkv_stride, rows, q_heads, rotary_dim, q_norm, k_norm, eps, inv_freq, positions,
                      row_sequence, row_slot, query, query_stride, key, key_stride, slot_positions, slot_stride};
  return launch_norm_rope_store(a, static_cast<cudaStream_t>(stream));
}

size_t qllm_k_decode_attention_workspace_bytes(const qllm_kv_batch* cache, uint32_t q_heads, int weights) {
  const char* who = "decode attention workspace";
  if (check_cache(cache, who) || check_page_geometry(cache, who) || check_query_heads(cache, q_heads)) return 0U;
  return decode_attention_workspace_bytes(*cache, q_heads, weights != 0);
}

int qllm_k_decode_attention(const qllm_kv_batch* cache, uint32_t row_type, const void* query, size_t query_stride,
                            const uint32_t* lengths, uint32_t q_heads, float scale, const float* weights_in,
                            float* weights_out, size_t weights_stride, void* out, size_t out_stride, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const char* who = "decode attention";
  int rc = check_cache(cache, who);
  if (rc || (rc = check_pages(cache, who)) || (rc = check_query_heads(cache, q_heads))) return rc;
  if (row_type > QLLM_ROW_F16 || !lengths || !workspace || !std::isfinite(scale))
    return fail(QLLM_INVALID_ARGUMENT, "invalid decode attention batch");
  if ((rc = check_words(who, lengths, weights_in, weights_out))) return rc;
  const size_t width = static_cast<size_t>(q_heads) * cache->head_dim, e = row_bytes(row_type);
  if (!rows_ok(query, cache->sequences, query_stride, row_type, width) || !rows_ok(out, cache->sequences, out_stride, row_type, width))
    return fail(QLLM_INVALID_ARGUMENT,
                "decode attention needs rows on 16-byte boundaries, strides that hold a row and are multiples of 16 bytes");
  if (overlap(Rows{query, cache->sequences, query_stride, width, e}, Rows{out, cache->sequences, out_stride, width, e}))
    return fail(QLLM_INVALID_ARGUMENT, "decode attention: query and out overlap");
  if (weights_in && !weights_out) return fail(QLLM_INVALID_ARGUMENT, "decode attention: weights_in without weights_out");
  if (weights_out) {
    if (weights_stride < kv_capacity(*cache) || !extent_ok(static_cast<size_t>(cache->sequences) * cache->kv_heads, weights_stride))
      return fail(QLLM_INVALID_ARGUMENT, "decode attention: the weights' stride does not hold every slot");
    const auto array = [&](const void* p) {
      return Rows{p, static_cast<size_t>(cache->sequences) * cache->kv_heads, weights_stride, kv_capacity(*cache), sizeof(float)};
    };
    if (weights_in && weights_in != weights_out && overlap(array(weights_in), array(weights_out)))
      return fail(QLLM_INVALID_ARGUMENT, "decode attention: weights overlap and are not in place");
  }
  if (!aligned(workspace, 16U) || workspace_bytes < decode_attention_workspace_bytes(*cache, q_heads, weights_out != nullptr))
    return fail(QLLM_INVALID_ARGUMENT, "decode attention workspace is too small or not on a 16-byte boundary");
  if ((rc = check_device(who, {cache->page_tables}, lengths))) return rc;
  DecodeAttentionArgs a{*cache, row_type, query, query_stride, lengths, q_heads, scale, weights_in, weights_out, weights_stride,
                        out, out_stride, workspace};
  return launch_decode_attention(a, static_cast<cudaStream_t>(stream));
}

size_t qllm_k_kv_evict_workspace_bytes(const qllm_kv_batch* cache, uint32_t budget) {
  const char* who = "KV eviction workspace";
  if (check_cache(cache, who) || check_page_geometry(cache, who)) return 0U;
  return kv_evict_workspace_bytes(*cache, budget);
}

int qllm_k_kv_evict(const qllm_kv_batch* cache, const uint32_t* lengths_in, uint32_t* lengths_out,
                    const uint32_t* next_positions, uint32_t budget, uint32_t recent, uint32_t sinks,
                    const float* weights_in, float* weights_out, const uint32_t* positions_in, uint32_t* positions_out,
                    size_t stride, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "KV eviction";
  int rc = check_cache(cache, who);
  if (rc || (rc = check_pages(cache, who))) return rc;
  if (!lengths_in || !lengths_out || !next_positions || !weights_in || !weights_out || !positions_in || !positions_out || !workspace)
    return fail(QLLM_INVALID_ARGUMENT, "invalid KV eviction batch");
  if ((rc = check_words(who, lengths_in, lengths_out, next_positions, weights_in, weights_out, positions_in, positions_out))) return rc;
  if (!budget || static_cast<uint64_t>(recent) + sinks > budget)
    return fail(QLLM_INVALID_ARGUMENT, "KV eviction needs a budget that holds the recent tokens and the sinks");
  if (stride < kv_capacity(*cache) || !extent_ok(static_cast<size_t>(cache->sequences) * cache->kv_heads, stride))
    return fail(QLLM_INVALID_ARGUMENT, "KV eviction: the stride does not hold every slot");
  const auto array = [&](const void* p) { return Rows{p, static_cast<size_t>(cache->sequences) * cache->kv_heads, stride, kv_capacity(*cache), 4U}; };
  if ((weights_in != weights_out && overlap(array(weights_in), array(weights_out))) ||
      (positions_in != positions_out && overlap(array(positions_in), array(positions_out))) ||
      overlap(array(weights_out), array(positions_in)) || overlap(array(weights_out), array(positions_out)) ||
      overlap(array(weights_in), array(positions_out)))
    return fail(QLLM_INVALID_ARGUMENT, "KV eviction: arrays overlap and are not in place");
  const size_t list = cache->sequences * sizeof(uint32_t);
  if ((lengths_in != lengths_out && overlap(lengths_in, list, lengths_out, list)) || overlap(next_positions, list, lengths_out, list))
    return fail(QLLM_INVALID_ARGUMENT, "KV eviction: arrays overlap and are not in place");
  if (!aligned(workspace, 16U) || workspace_bytes < kv_evict_workspace_bytes(*cache, budget))
    return fail(QLLM_INVALID_ARGUMENT, "KV eviction workspace is too small or not on a 16-byte boundary");
  if ((rc = check_device(who, {cache->page_tables}, lengths_in))) return rc;
  KvEvictArgs a{*cache, lengths_in, lengths_out, next_positions, budget, recent, sinks, weights_in, weights_out, positions_in,
                positions_out, stride, workspace};
  return launch_kv_evict(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
