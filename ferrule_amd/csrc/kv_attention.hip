// Attention over the MXFP4 key/value cache (no reference symbol; formats, layout and batch
// description: include/ferrule_hip_provider.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ferrule_hip_provider.h"
#include "kv_cache.cuh"

namespace ferrule_hip {
namespace {

constexpr uint32_t kChunk = 256;  // tokens that a workgroup scores at a time, one per thread

__device__ __forceinline__ float load_query(uint64_t q, uint64_t at, bool f32) {
  return f32 ? bf16_round(global_ptr<const float>(q)[at]) : bf16_bits_to_f32(global_ptr<const uint16_t>(q)[at]);
}

__device__ __forceinline__ float block_value(uint32_t nibble, uint32_t byte) {
  return byte == kNanBlock ? __uint_as_float(0x7fc00000u) : fp4_e2m1_decode(nibble) * e8m0_to_f32(byte);
}

// One workgroup per row and query head: a thread scores one token, then owns values of the row.
template <uint32_t D>
__global__ __launch_bounds__(256) void kv_attention_row_kernel(FerruleHipKvAttentionArgs a) {
  using Layout = KvLayout<D>;
  __shared__ float query[D];
  __shared__ float weight[kChunk];
  __shared__ int32_t page_of[kChunk];
  __shared__ float reduce[8];
  const uint32_t b = blockIdx.y, thread = threadIdx.x;
  const uint32_t head = blockIdx.x % a.q_heads, index = blockIdx.x / a.q_heads;
  const KvSequence s = kv_sequence(a.query_indptr, a.sequence_lengths, b, a.rows, a.max_query_length);
  if (s.bad && blockIdx.x == 0u && thread == 0u) kv_report(a.error);
  if (index >= s.rows) return;
  const uint32_t kv_head = head / (a.q_heads / a.kv_heads);
  const uint64_t row = s.row + static_cast<uint64_t>(index);
  const bool f32_query = (a.flags & FERRULE_HIP_KV_ATTENTION_QUERY_F32) != 0u;
  for (uint32_t d = thread; d < D; d += 256u) {
    query[d] = load_query(a.q, row * a.q_row_stride + head * a.q_head_stride + d, f32_query);
  }
  __syncthreads();
  const int32_t position = s.position + static_cast<int32_t>(index);
  // validate() keeps the table below 2^31 tokens
  const int32_t last = min(position, static_cast<int32_t>(a.max_pages * a.page_tokens) - 1);
  if (last < position && thread == 0u) kv_report(a.error);
  float top = -INFINITY, total = 0.0f;
  constexpr uint32_t kOwn = D > 256u ? D / 256u : 1u;  // values of the row per thread
  float sum[kOwn] = {};
  for (int32_t begin = 0; begin <= last; begin += static_cast<int32_t>(kChunk)) {
    if (a.window != 0u && position - (begin + static_cast<int32_t>(kChunk) - 1) >= static_cast<int32_t>(a.window) &&
        begin >= static_cast<int32_t>(a.sinks)) {
      continue;  // nothing of the chunk is seen
    }
    const int32_t j = begin + static_cast<int32_t>(thread);
    bool seen = j <= last && (a.window == 0u || static_cast<uint32_t>(position - j) < a.window ||
                                  static_cast<uint32_t>(j) < a.sinks);
    int32_t page = -1;
    if (seen) {
      const uint32_t slot = static_cast<uint32_t>(j) / a.page_tokens;
      page = global_ptr<const int32_t>(a.page_table)[static_cast<uint64_t>(b) * a.max_pages + slot];
      if (static_cast<uint32_t>(page) >= a.page_count) {
        page = -1;
        seen = false;
        kv_report(a.error);
      }
    }
    float score = -INFINITY;
    if (seen) {
      const uint64_t page_head = static_cast<uint64_t>(page) * a.kv_heads + kv_head;
      const uint32_t t = static_cast<uint32_t>(j) % a.page_tokens;
      const uint8_t *payload = global_ptr<const uint8_t>(a.k_payload) + Layout::payload(page_head, a.page_tokens);
      const uint8_t *scales = global_ptr<const uint8_t>(a.k_scales) + Layout::scales(page_head, a.page_tokens);
      float dot = 0.0f;
      for (uint32_t d = 0; d < D; d += 2u) {
        const uint32_t byte = payload[Layout::key_byte(t, d / 128u) + (d % 128u) / 2u];
        const uint32_t scale = scales[Layout::key_scale(t, d / 32u)];
        dot += query[d] * block_value(byte & 15u, scale) + query[d + 1u] * block_value(byte >> 4, scale);
      }
      score = dot * a.softmax_scale;
    }
    float chunk_top = wave_max(score);  // a NaN score is caught by its weight
    if ((thread & 63u) == 0u) reduce[thread >> 6] = chunk_top;
    __syncthreads();
    chunk_top = fmaxf(fmaxf(reduce[0], reduce[1]), fmaxf(reduce[2], reduce[3]));
    const float next = fmaxf(top, chunk_top);
    const float shift = next == -INFINITY ? 0.0f : next;
    const float w = seen ? expf(score - shift) : 0.0f;
    weight[thread] = w;
    page_of[thread] = seen ? page : -1;
    const float wave_total = wave_sum(w);
    if ((thread & 63u) == 0u) reduce[4 + (thread >> 6)] = wave_total;
    __syncthreads();
    const float keep = top == -INFINITY ? 0.0f : expf(top - shift);
    total = total * keep + ((reduce[4] + reduce[5]) + (reduce[6] + reduce[7]));
    top = next;
    for (uint32_t i = 0; i < kOwn; ++i) {
      const uint32_t d = thread + i * 256u;
      if (d >= D) break;
      float acc = sum[i] * keep;
      for (uint32_t u = 0; u < kChunk; ++u) {
        if (page_of[u] < 0) continue;
        const uint64_t page_head = static_cast<uint64_t>(page_of[u]) * a.kv_heads + kv_head;
        const uint32_t t = static_cast<uint32_t>(begin + static_cast<int32_t>(u)) % a.page_tokens;
        const uint32_t byte =
            (global_ptr<const uint8_t>(a.v_payload) + Layout::payload(page_head, a.page_tokens))[Layout::value_byte(t, d / 2u)];
        const uint32_t scale =
            (global_ptr<const uint8_t>(a.v_scales) + Layout::scales(page_head, a.page_tokens))[Layout::value_scale(t, d / 32u)];
        acc += weight[u] * block_value((d & 1u) ? byte >> 4 : byte & 15u, scale);
      }
      sum[i] = acc;
    }
    __syncthreads();
  }
  for (uint32_t i = 0; i < kOwn; ++i) {
    const uint32_t d = thread + i * 256u;
    if (d >= D) break;
    const float o = top == -INFINITY && total == 0.0f ? 0.0f : sum[i] / total;
    const uint64_t at = row * a.output_row_stride + head * a.output_head_stride + d;
    if (a.flags & FERRULE_HIP_KV_ATTENTION_OUTPUT_F32) {
      global_ptr<float>(a.output)[at] = o;
    } else {
      global_ptr<uint16_t>(a.output)[at] = bf16_rne_bits(o);
    }
  }
}

// Scalar fields and strides; pointers are looked at by validate().
FerruleHipStatus validate_shape(const FerruleHipKvAttentionArgs &a) {
  if (a.q_heads == 0u || a.kv_heads == 0u || a.q_heads % a.kv_heads != 0u || a.head_dim == 0u || a.page_count == 0u ||
      a.max_pages == 0u || a.max_query_length == 0u || !kv_page_tokens_valid(a.page_tokens) ||
      a.page_count > 0x7fffffffu || a.rows > 0x7fffffffu || a.window > 0x7fffffffu || a.sinks > 0x7fffffffu ||
      (a.flags & ~(FERRULE_HIP_KV_ATTENTION_QUERY_F32 | FERRULE_HIP_KV_ATTENTION_OUTPUT_F32)) != 0u ||
      !(a.softmax_scale > 0.0f && a.softmax_scale <= 3.4028234e38f)) {
    return FERRULE_HIP_INVALID_ARGUMENT;
  }
  if (!kv_head_dim_supported(a.head_dim)) return FERRULE_HIP_UNSUPPORTED;
  if (static_cast<uint64_t>(a.max_pages) * a.page_tokens > 0x7fffffffull) return FERRULE_HIP_UNSUPPORTED;
  if (a.batch > 65535u || static_cast<uint64_t>(a.max_query_length) * a.q_heads > 0x7fffffffull) return FERRULE_HIP_UNSUPPORTED;
  return FERRULE_HIP_SUCCESS;
}

FerruleHipStatus validate(const FerruleHipKvAttentionArgs &a) {
  if (a.batch == 0u || a.rows == 0u) return FERRULE_HIP_SUCCESS;  // nothing to do
  const FerruleHipStatus status = validate_shape(a);
  if (status == FERRULE_HIP_INVALID_ARGUMENT) return status;
  const uint32_t q_bytes = (a.flags & FERRULE_HIP_KV_ATTENTION_QUERY_F32) ? 4u : 2u;
  const uint32_t o_bytes = (a.flags & FERRULE_HIP_KV_ATTENTION_OUTPUT_F32) ? 4u : 2u;
  if (!kv_rows_aligned(a.q, a.q_row_stride, a.q_head_stride, q_bytes) ||
      !kv_rows_aligned(a.output, a.output_row_stride, a.output_head_stride, o_bytes) || !kv_aligned16(a.k_payload) ||
      !kv_aligned16(a.k_scales) || !kv_aligned16(a.v_payload) || !kv_aligned16(a.v_scales) || a.query_indptr == 0u ||
      a.sequence_lengths == 0u || a.page_table == 0u || ((a.query_indptr | a.sequence_lengths | a.page_table | a.error) & 3u)) {
    return FERRULE_HIP_INVALID_ARGUMENT;
  }
  const uint64_t needed = ferrule_hip_kv_attention_workspace_size(&a);
  if (needed != 0u && (a.workspace == 0u || (a.workspace & 255u) != 0u || a.workspace_bytes < needed)) {
    return FERRULE_HIP_INVALID_ARGUMENT;
  }
  return status;
}

template <uint32_t D>
void launch(const FerruleHipKvAttentionArgs &a, hipStream_t stream) {
  const uint32_t rows = a.max_query_length < a.rows ? a.max_query_length : a.rows;
  kv_attention_row_kernel<D><<<dim3(rows * a.q_heads, a.batch), 256, 0, stream>>>(a);
}

}  // namespace
}  // namespace ferrule_hip

extern "C" uint64_t ferrule_hip_kv_attention_workspace_size(const FerruleHipKvAttentionArgs *args) {
  (void)args;
  return 0;
}

extern "C" int32_t ferrule_hip_kv_attention_can_implement(const FerruleHipKvAttentionArgs *args) {
  return args == nullptr ? FERRULE_HIP_INVALID_ARGUMENT : ferrule_hip::validate(*args);
}

extern "C" int32_t ferrule_hip_kv_attention_launch(const FerruleHipKvAttentionArgs *args) {
  using namespace ferrule_hip;
  if (args == nullptr) return FERRULE_HIP_INVALID_ARGUMENT;
  const FerruleHipStatus status = validate(*args);
  if (status != FERRULE_HIP_SUCCESS || args->batch == 0u || args->rows == 0u) return status;
  const FerruleHipKvAttentionArgs &a = *args;
  hipStream_t stream = reinterpret_cast<hipStream_t>(static_cast<uintptr_t>(a.stream));
  clear_launch_error();
  switch (a.head_dim) {
    case 64: launch<64>(a, stream); break;
    case 128: launch<128>(a, stream); break;
    case 256: launch<256>(a, stream); break;
    default: launch<512>(a, stream); break;
  }
  return take_launch_error() == hipSuccess ? FERRULE_HIP_SUCCESS : FERRULE_HIP_LAUNCH_FAILED;
}
