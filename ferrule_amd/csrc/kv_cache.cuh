// Addressing of the MXFP4 key/value cache and of a batch's rows, shared by kv_cache.hip and
// kv_attention.hip (layout and batch description: include/ferrule_hip_provider.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "numeric.cuh"

namespace ferrule_hip {

constexpr uint32_t kNanBlock = 255u;  // scale byte of a block that held an infinity or a NaN

// Rows of one sequence.  Row numbers are clamped to what the row tensors hold, so that a bad index or
// count cannot lead outside them; positions are checked against the table where they are followed.
struct KvSequence {
  uint32_t row;      // first row of the sequence
  uint32_t rows;     // its new rows
  int32_t position;  // position of its first new row, negative when it has fewer tokens than rows
  bool bad;          // something was clamped
};

// Metadata that nothing writes while the kernel runs, at a wave-uniform index: through the constant
// address space it is a scalar load, which is counted apart from the vector loads in flight - as a
// vector load its wait would drain them.
__device__ __forceinline__ int32_t kv_uniform(uint64_t address, uint64_t index) {
  typedef __attribute__((address_space(4))) const int32_t constant_t;
  return reinterpret_cast<constant_t *>(static_cast<uintptr_t>(address))[index];
}

__device__ __forceinline__ KvSequence kv_sequence_of(int32_t first, int32_t last, int32_t length, uint32_t rows,
                                                     uint32_t max_query_length) {
  KvSequence s;
  const int32_t row = min(max(first, 0), static_cast<int32_t>(rows));
  const int32_t end = min(max(last, row), static_cast<int32_t>(rows));
  s.row = static_cast<uint32_t>(row);
  s.rows = static_cast<uint32_t>(end - row);
  s.position = max(length, 0) - static_cast<int32_t>(s.rows);
  s.bad = row != first || end != last || length < 0 || s.rows > max_query_length;
  if (s.rows > max_query_length) s.rows = max_query_length;  // the rows that the grid covers
  return s;
}

__device__ __forceinline__ KvSequence kv_sequence(uint64_t query_indptr, uint64_t sequence_lengths, uint32_t b,
                                                  uint32_t rows, uint32_t max_query_length) {
  return kv_sequence_of(kv_uniform(query_indptr, b), kv_uniform(query_indptr, b + 1u), kv_uniform(sequence_lengths, b), rows,
                        max_query_length);
}

// What one wave wrote to LDS, read by its other lanes: the wave's LDS operations run in order, only
// the compiler has to keep them so.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ void kv_report(uint64_t error) {
  if (error != 0u) *global_ptr<int32_t>(error) = 1;
}

// Byte offsets of one (page, head): token offsets inside it are added by the callers.
template <uint32_t D>
struct KvLayout {
  static constexpr uint32_t kBlocks = D / 32u;                      // scale blocks of a row
  static constexpr uint32_t kKeyChunks = (D + 127u) / 128u;         // 128-value pieces of a key row
  static constexpr uint32_t kKeyBytes = (D < 128u ? D : 128u) / 2u; // payload bytes of one piece
  // token t of a page's head
  static __device__ __forceinline__ uint64_t payload(uint64_t page_head, uint32_t page_tokens) {
    return page_head * page_tokens * (D / 2u);
  }
  static __device__ __forceinline__ uint64_t scales(uint64_t page_head, uint32_t page_tokens) {
    return page_head * page_tokens * kBlocks;
  }
  static __device__ __forceinline__ uint32_t key_byte(uint32_t t, uint32_t chunk) {
    return (t & ~31u) * (D / 2u) + chunk * 32u * kKeyBytes + (t & 31u) * kKeyBytes;
  }
  static __device__ __forceinline__ uint32_t key_scale(uint32_t t, uint32_t block) {
    return (t & ~31u) * kBlocks + block * 32u + (t & 31u);
  }
  static __device__ __forceinline__ uint32_t value_byte(uint32_t t, uint32_t pair) {
    return (t & ~7u) * (D / 2u) + pair * 8u + (t & 7u);
  }
  static __device__ __forceinline__ uint32_t value_scale(uint32_t t, uint32_t block) {
    return (t & ~7u) * kBlocks + block * 8u + (t & 7u);
  }
};

// Host: what all three operators refuse about the cache and the batch.
inline bool kv_aligned16(uint64_t p) { return p != 0u && (p & 15u) == 0u; }
inline bool kv_head_dim_supported(uint32_t d) { return d == 64u || d == 128u || d == 256u || d == 512u; }
inline bool kv_page_tokens_valid(uint32_t p) { return p >= 32u && p <= 1024u && (p & (p - 1u)) == 0u; }
// a strided row tensor: every row of every head on 16 bytes (a stride that takes nothing anywhere may be any)
inline bool kv_rows_aligned(uint64_t base, uint32_t rows, uint64_t row_stride, uint32_t heads, uint64_t head_stride, uint32_t value_bytes) {
  return kv_aligned16(base) && (rows == 1u || (row_stride * value_bytes) % 16u == 0u) &&
         (heads == 1u || (head_stride * value_bytes) % 16u == 0u);
}

}  // namespace ferrule_hip
