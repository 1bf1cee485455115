// Writing the MXFP4 key/value cache and reading it back (no reference symbol; formats, layout and
// batch description: include/ferrule_hip_provider.h).
//
// Both kernels move a row's bytes once and are bound by memory for whole prompts, by launch and latency
// for a decode step's rows.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ferrule_hip_provider.h"
#include "kv_cache.cuh"

namespace ferrule_hip {
namespace {

constexpr uint32_t kWaves = 4;
constexpr uint32_t kTokens = 32;  // of a tile

// Where a wave works: 32 neighbouring tokens of one head.  In two steps, since rows can be asked for before the page
// is known.
struct KvTile {
  KvSequence sequence;
  uint32_t head;
  int32_t offset;       // row of the sequence of the tile's first token, may be negative
  uint32_t page_token;  // of that token
  uint64_t page_head;   // page * kv_heads + head
  bool page_valid;      // false: no token of the tile has a place

  // Tile `index` of sequence blockIdx.y, by head first; false when the sequence has no such tile.
  __device__ __forceinline__ bool rows_of(const FerruleHipKvCacheArgs &a, uint32_t index) {
    head = index % a.kv_heads;
    const uint32_t group = index / a.kv_heads;
    sequence = kv_sequence(a.query_indptr, a.sequence_lengths, blockIdx.y, a.rows, a.max_query_length);
    if (sequence.bad && index == 0u && (threadIdx.x & 63u) == 0u) kv_report(a.error);
    // tiles are counted from the one that holds the first row; its position may be negative
    const uint32_t before = static_cast<uint32_t>(sequence.position) & (kTokens - 1u);
    if (group * kTokens >= before + sequence.rows) return false;
    offset = static_cast<int32_t>(group * kTokens - before);
    return true;
  }
  __device__ __forceinline__ void page_of(const FerruleHipKvCacheArgs &a) {
    const int32_t first = sequence.position + offset;
    page_valid = false;
    page_head = 0;
    page_token = 0;
    const uint32_t slot = static_cast<uint32_t>(first) / a.page_tokens;
    if (first >= 0 && slot < a.max_pages) {
      const int32_t page = kv_uniform(a.page_table, static_cast<uint64_t>(blockIdx.y) * a.max_pages + slot);
      page_token = static_cast<uint32_t>(first) % a.page_tokens;
      page_valid = static_cast<uint32_t>(page) < a.page_count;
      if (page_valid) page_head = static_cast<uint64_t>(page) * a.kv_heads + head;
    }
    if (!page_valid && (threadIdx.x & 63u) == 0u) kv_report(a.error);
  }
};

// Eight consecutive values of a row as f32.
__device__ __forceinline__ void load8(const uint16_t *src, float (&x)[8]) {
  const i32x4_t w = *reinterpret_cast<const i32x4_t *>(src);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __uint_as_float(static_cast<uint32_t>(w[e]) << 16);
    x[2 * e + 1] = __uint_as_float(static_cast<uint32_t>(w[e]) & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const float *src, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x4_t w = reinterpret_cast<const f32x4_t *>(src)[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[4 * i + e] = w[e];
  }
}

// A quarter of a scale block (8 values; lanes ^ 1, 2, 3 have the others) -> its four payload bytes and
// the block's scale byte.  All in bits: with amax = 1.f * 2^e the smallest n with 6 * 2^n >= amax is
// e - 2 while 1.f <= 1.5, else e - 1; and |x| / 2^n rounds to the one-mantissa-bit grid by adding
// just under half a step, which sends a tie down.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t &packed) {
  uint32_t top = 0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1, 64)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2, 64)));
  packed = 0u;
  if (top >= 0x7f800000u) return kNanBlock;
  const int32_t exponent = static_cast<int32_t>(top >> 23) - 127;
  int32_t n = exponent - 2 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0);
  n = max(n, -126);
  const float inverse = __uint_as_float(static_cast<uint32_t>(127 - n) << 23);  // n <= 126: normal
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = x[i] * inverse;  // exact, |q| <= 6, or below every threshold
    const uint32_t bits = __float_as_uint(q) & 0x7fffffffu;
    const float m = __uint_as_float(bits);
    const uint32_t large = ((bits + 0x1fffffu) >> 22) - 252u;            // m >= 1: 2..7
    const uint32_t small = (m > 0.25f ? 1u : 0u) + (m > 0.75f ? 1u : 0u);  // m < 1: 0..2
    const uint32_t code = (m >= 1.0f ? large : small) | ((__float_as_uint(q) >> 28) & 8u);
    packed |= code << (4 * i);
  }
  return static_cast<uint32_t>(n + 127);
}

// A wave has up to 128 values of one head of eight neighbouring tokens, the unit of the value layout, and a workgroup
// those of 32 tokens: the scale bytes of a cache line come from one place.  A lane takes eight values, so that 128 of
// a row are sixteen lanes side by side, and keys and values are asked for together, before the page is known: a decode
// step's rows are a chain of memory latencies.
template <typename T, uint32_t D>
__global__ __launch_bounds__(256) void kv_append_kernel(FerruleHipKvCacheArgs a) {
  using Layout = KvLayout<D>;
  constexpr uint32_t kLanes = (D < 128u ? D : 128u) / 8u;  // of a row
  constexpr uint32_t kTogether = 64u / kLanes;             // rows side by side: 4, or 8 at D = 64
  constexpr uint32_t kPasses = 8u / kTogether;
  // the bytes of 128 values of eight tokens, turned in LDS: [value pair][token]
  __shared__ __align__(16) uint8_t turned[kWaves][64][8];
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t c = blockIdx.x % Layout::kKeyChunks;  // 128-value piece of the rows
  KvTile tile;
  if (!tile.rows_of(a, blockIdx.x / Layout::kKeyChunks)) return;
  const uint32_t column = lane % kLanes, part = lane / kLanes;
  const int32_t offset = tile.offset + static_cast<int32_t>(8u * wave);
  const int32_t rows = static_cast<int32_t>(tile.sequence.rows);
  const bool any = offset < rows && offset > -8;
  const bool whole = offset >= 0 && offset + 8 <= rows;
  float k[kPasses][8], v[kPasses][8];
  bool live[kPasses];
  if (any) {
    const T *keys = global_ptr<const T>(a.keys) + tile.head * a.key_head_stride + c * 128u + column * 8u;
    const T *values = global_ptr<const T>(a.values) + tile.head * a.value_head_stride + c * 128u + column * 8u;
#pragma unroll
    for (uint32_t p = 0; p < kPasses; ++p) {
      const int32_t row = offset + static_cast<int32_t>(p * kTogether + part);
      live[p] = row >= 0 && row < rows;
      // a row that is not there is read as one that is: its bytes are not written
      const uint64_t at = tile.sequence.row + static_cast<uint64_t>(live[p] ? row : max(offset, 0));
      load8(keys + at * a.key_row_stride, k[p]);
      load8(values + at * a.value_row_stride, v[p]);
    }
  }
  tile.page_of(a);
  if (!any || !tile.page_valid) return;
  const uint32_t first = tile.page_token + 8u * wave;
  uint8_t *k_payload = global_ptr<uint8_t>(a.k_payload) + Layout::payload(tile.page_head, a.page_tokens);
  uint8_t *k_scales = global_ptr<uint8_t>(a.k_scales) + Layout::scales(tile.page_head, a.page_tokens);
  uint8_t *v_payload = global_ptr<uint8_t>(a.v_payload) + Layout::payload(tile.page_head, a.page_tokens);
  uint8_t *v_scales = global_ptr<uint8_t>(a.v_scales) + Layout::scales(tile.page_head, a.page_tokens);
#pragma unroll
  for (uint32_t p = 0; p < kPasses; ++p) {
    const uint32_t t = p * kTogether + part, token = first + t, block = c * 4u + column / 4u;
    uint32_t kq, vq;
    const uint32_t ks = quantise8(k[p], kq);
    const uint32_t vs = quantise8(v[p], vq);
    if (live[p]) {
      *reinterpret_cast<uint32_t *>(k_payload + Layout::key_byte(token, c) + column * 4u) = kq;
      if ((column & 3u) == 0u) {
        k_scales[Layout::key_scale(token, block)] = static_cast<uint8_t>(ks);
        v_scales[Layout::value_scale(token, block)] = static_cast<uint8_t>(vs);
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
      const uint8_t byte = static_cast<uint8_t>(vq >> (8u * i));
      if (whole) {  // wave-uniform
        turned[wave][column * 4u + i][t] = byte;
      } else if (live[p]) {
        v_payload[Layout::value_byte(token, c * 64u + column * 4u + i)] = byte;
      }
    }
  }
  if (whole) {
    wave_lds_fence();
    const uint2 pair = *reinterpret_cast<const uint2 *>(&turned[wave][lane][0]);
    if (c * 64u + lane < D / 2u) {
      *reinterpret_cast<uint2 *>(v_payload + Layout::value_byte(first, c * 64u + lane)) = pair;
    }
  }
}

// Eight values of a row from four payload bytes (values 0, 1 in the low byte) and their scale byte.
__device__ __forceinline__ void expand8(uint32_t bytes, uint32_t scale_byte, float (&x)[8]) {
  // 2^(byte - 127); 255 is a block of NaN.  The converter's scale is an f32 exponent field, which has no 2^-127:
  // a byte of 0 (which the writer never writes) goes through the product below instead.
  const float scale = scale_byte == kNanBlock ? __uint_as_float(0x7fc00000u) : e8m0_to_f32(scale_byte);
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    f32x2_t v;
    // the byte is an immediate of the instruction
    if (p == 0) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(bytes, 1.0f, 0);
    if (p == 1) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(bytes, 1.0f, 1);
    if (p == 2) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(bytes, 1.0f, 2);
    if (p == 3) v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(bytes, 1.0f, 3);
    x[2 * p] = v[0] * scale;
    x[2 * p + 1] = v[1] * scale;
  }
}

__device__ __forceinline__ void store8(float *dst, const float (&x)[8]) {
  const f32x4_t lo = {x[0], x[1], x[2], x[3]}, hi = {x[4], x[5], x[6], x[7]};
  __builtin_nontemporal_store(lo, reinterpret_cast<f32x4_t *>(dst));
  __builtin_nontemporal_store(hi, reinterpret_cast<f32x4_t *>(dst) + 1);
}
__device__ __forceinline__ void store8(uint16_t *dst, const float (&x)[8]) {  // exact in BF16
  i32x4_t w;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    w[p] = static_cast<int>((__float_as_uint(x[2 * p]) >> 16) | (__float_as_uint(x[2 * p + 1]) & 0xffff0000u));
  }
  __builtin_nontemporal_store(w, reinterpret_cast<i32x4_t *>(dst));
}

// A wave has the keys, or the values, of one head of 32 neighbouring tokens: a lane takes eight values
// at a time, so that it stores 16 (BF16) or 32 bytes and a row is D / 8 lanes side by side, past the caches:
// the rows are more than they hold.  4 sequences of up to 8192 tokens, 8 heads of 128: 17.6 us, 6.0 TB/s
// (24.3 us with ordinary stores, 45 us with two values a lane and store).
template <typename T, uint32_t D>
__global__ __launch_bounds__(256) void kv_read_kernel(FerruleHipKvCacheArgs a) {
  using Layout = KvLayout<D>;
  constexpr uint32_t kLanes = D / 8u;       // of a row
  constexpr uint32_t kTogether = 64u / kLanes;  // rows (keys) or groups of eight tokens (values) side by side
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
  const bool values = (wave & 1u) != 0u;
  KvTile tile;
  if (!tile.rows_of(a, wave >> 1)) return;
  tile.page_of(a);
  const uint32_t column = lane % kLanes, part = lane / kLanes;
  const int32_t offset = tile.offset;
  const int32_t rows = static_cast<int32_t>(tile.sequence.rows);
  const uint32_t block = column / 4u;
  if (!values) {
    const uint8_t *payload = global_ptr<const uint8_t>(a.k_payload) + Layout::payload(tile.page_head, a.page_tokens);
    const uint8_t *scales = global_ptr<const uint8_t>(a.k_scales) + Layout::scales(tile.page_head, a.page_tokens);
    T *out = global_ptr<T>(a.keys) + tile.head * a.key_head_stride + column * 8u;
    constexpr uint32_t kAtOnce = 8u;  // loads in flight
#pragma unroll 1
    for (uint32_t first = part; first < 32u; first += kAtOnce * kTogether) {
      uint32_t bytes[kAtOnce], scale[kAtOnce];
#pragma unroll
      for (uint32_t k = 0; k < kAtOnce; ++k) {
        const uint32_t token = tile.page_token + min(first + k * kTogether, 31u);
        bytes[k] = *reinterpret_cast<const uint32_t *>(payload + Layout::key_byte(token, column / 16u) + (column % 16u) * 4u);
        scale[k] = scales[Layout::key_scale(token, block)];
      }
#pragma unroll
      for (uint32_t k = 0; k < kAtOnce; ++k) {
        const uint32_t t = first + k * kTogether;
        const int32_t index = offset + static_cast<int32_t>(t);
        if (t >= 32u || index < 0 || index >= rows) continue;
        float x[8];
        expand8(tile.page_valid ? bytes[k] : 0u, tile.page_valid ? scale[k] : 127u, x);
        store8(out + (tile.sequence.row + static_cast<uint64_t>(index)) * a.key_row_stride, x);
      }
    }
    return;
  }
  const uint8_t *payload = global_ptr<const uint8_t>(a.v_payload) + Layout::payload(tile.page_head, a.page_tokens);
  const uint8_t *scales = global_ptr<const uint8_t>(a.v_scales) + Layout::scales(tile.page_head, a.page_tokens);
  T *out = global_ptr<T>(a.values) + tile.head * a.value_head_stride + column * 8u;
#pragma unroll
  for (uint32_t eight = 0; eight < 32u; eight += 8u * kTogether) {
    const uint32_t first = eight + 8u * part;
    if (first >= 32u) break;
    // four pairs of values of eight tokens: [pair][token]
    const uint2 *src = reinterpret_cast<const uint2 *>(payload + Layout::value_byte(tile.page_token + first, column * 4u));
    const uint2 pair[4] = {src[0], src[1], src[2], src[3]};
    const uint2 scale = *reinterpret_cast<const uint2 *>(scales + Layout::value_scale(tile.page_token + first, block));
#pragma unroll
    for (uint32_t t = 0; t < 8u; ++t) {
      const int32_t index = offset + static_cast<int32_t>(first + t);
      if (index < 0 || index >= rows) continue;
      // byte t of every pair
      const uint32_t sel = 0x0c0c0000u | (4u + (t & 3u)) << 8 | (t & 3u);
      const uint32_t lo = __builtin_amdgcn_perm(t < 4u ? pair[1].x : pair[1].y, t < 4u ? pair[0].x : pair[0].y, sel);
      const uint32_t hi = __builtin_amdgcn_perm(t < 4u ? pair[3].x : pair[3].y, t < 4u ? pair[2].x : pair[2].y, sel);
      const uint32_t scale_byte = ((t < 4u ? scale.x : scale.y) >> (8u * (t & 3u))) & 255u;
      float x[8];
      expand8(tile.page_valid ? lo | (hi << 16) : 0u, tile.page_valid ? scale_byte : 127u, x);
      store8(out + (tile.sequence.row + static_cast<uint64_t>(index)) * a.value_row_stride, x);
    }
  }
}

// Tiles that some rows of a sequence can touch, starting at the last token of one.
uint32_t tiles_of(uint32_t rows) { return rows / kTokens + (rows % kTokens + kTokens - 2u) / kTokens + 1u; }

FerruleHipStatus validate(const FerruleHipKvCacheArgs &a) {
  if (a.batch == 0u || a.rows == 0u) return FERRULE_HIP_SUCCESS;  // nothing to do
  if (a.reserved != 0u || a.value_type > FERRULE_HIP_KV_BF16) return FERRULE_HIP_INVALID_ARGUMENT;
  if (a.kv_heads == 0u || a.head_dim == 0u || a.page_count == 0u || a.max_pages == 0u || a.max_query_length == 0u ||
      !kv_page_tokens_valid(a.page_tokens) || a.page_count > 0x7fffffffu || a.rows > 0x7fffffffu) {
    return FERRULE_HIP_INVALID_ARGUMENT;
  }
  const uint32_t bytes = a.value_type == FERRULE_HIP_KV_BF16 ? 2u : 4u;
  if (!kv_rows_aligned(a.keys, a.rows, a.key_row_stride, a.kv_heads, a.key_head_stride, bytes) ||
      !kv_rows_aligned(a.values, a.rows, a.value_row_stride, a.kv_heads, a.value_head_stride, bytes) ||
      !kv_aligned16(a.k_payload) || !kv_aligned16(a.k_scales) || !kv_aligned16(a.v_payload) || !kv_aligned16(a.v_scales) || a.query_indptr == 0u ||
      a.sequence_lengths == 0u || a.page_table == 0u || ((a.query_indptr | a.sequence_lengths | a.page_table | a.error) & 3u)) {
    return FERRULE_HIP_INVALID_ARGUMENT;
  }
  if (!kv_head_dim_supported(a.head_dim)) return FERRULE_HIP_UNSUPPORTED;
  // batch in the grid's y; the threads of x, 256 for each head of a tile and 128 values of it at most, count in 32 bits
  const uint64_t workgroups = static_cast<uint64_t>(tiles_of(a.max_query_length)) * a.kv_heads * ((a.head_dim + 127u) / 128u);
  if (a.batch > 65535u || workgroups > 0xffffffull) {
    return FERRULE_HIP_UNSUPPORTED;
  }
  return FERRULE_HIP_SUCCESS;
}

// Rows that read writes stand once each; this is what shows it without a look at every row.
FerruleHipStatus validate_read(const FerruleHipKvCacheArgs &a) {
  const FerruleHipStatus status = validate(a);
  if (status == FERRULE_HIP_INVALID_ARGUMENT || a.batch == 0u || a.rows == 0u) return status;
  const bool rows = a.rows > 1u && (a.key_row_stride == 0u || a.value_row_stride == 0u);
  const bool heads = a.kv_heads > 1u && (a.key_head_stride == 0u || a.value_head_stride == 0u);
  return rows || heads || a.keys == a.values ? FERRULE_HIP_INVALID_ARGUMENT : status;
}

template <template <typename, uint32_t> class Launch>
FerruleHipStatus dispatch(const FerruleHipKvCacheArgs *args) {
  if (args == nullptr) return FERRULE_HIP_INVALID_ARGUMENT;
  const FerruleHipStatus status = Launch<float, 64>::check(*args);
  if (status != FERRULE_HIP_SUCCESS || args->batch == 0u || args->rows == 0u) return status;
  const FerruleHipKvCacheArgs &a = *args;
  hipStream_t stream = reinterpret_cast<hipStream_t>(static_cast<uintptr_t>(a.stream));
  const uint32_t tiles = tiles_of(a.max_query_length < a.rows ? a.max_query_length : a.rows);
  const dim3 grid((tiles * a.kv_heads * Launch<float, 64>::waves_per_tile(a.head_dim) + kWaves - 1u) / kWaves, a.batch);
  clear_launch_error();
  if (a.value_type == FERRULE_HIP_KV_BF16) {
    switch (a.head_dim) {
      case 64: Launch<uint16_t, 64>::run(a, grid, stream); break;
      case 128: Launch<uint16_t, 128>::run(a, grid, stream); break;
      case 256: Launch<uint16_t, 256>::run(a, grid, stream); break;
      default: Launch<uint16_t, 512>::run(a, grid, stream); break;
    }
  } else {
    switch (a.head_dim) {
      case 64: Launch<float, 64>::run(a, grid, stream); break;
      case 128: Launch<float, 128>::run(a, grid, stream); break;
      case 256: Launch<float, 256>::run(a, grid, stream); break;
      default: Launch<float, 512>::run(a, grid, stream); break;
    }
  }
  return take_launch_error() == hipSuccess ? FERRULE_HIP_SUCCESS : FERRULE_HIP_LAUNCH_FAILED;
}

template <typename T, uint32_t D>
struct Append {
  static FerruleHipStatus check(const FerruleHipKvCacheArgs &a) { return validate(a); }
  // eight tokens and up to 128 values each
  static uint32_t waves_per_tile(uint32_t head_dim) { return 4u * ((head_dim + 127u) / 128u); }
  static void run(const FerruleHipKvCacheArgs &a, dim3 grid, hipStream_t stream) {
    kv_append_kernel<T, D><<<grid, 256, 0, stream>>>(a);
  }
};
template <typename T, uint32_t D>
struct Read {
  static FerruleHipStatus check(const FerruleHipKvCacheArgs &a) { return validate_read(a); }
  static uint32_t waves_per_tile(uint32_t) { return 2u; }  // keys and values
  static void run(const FerruleHipKvCacheArgs &a, dim3 grid, hipStream_t stream) {
    kv_read_kernel<T, D><<<grid, 256, 0, stream>>>(a);
  }
};

}  // namespace
}  // namespace ferrule_hip

extern "C" int32_t ferrule_hip_kv_cache_append_can_implement(const FerruleHipKvCacheArgs *args) {
  return args == nullptr ? FERRULE_HIP_INVALID_ARGUMENT : ferrule_hip::validate(*args);
}
extern "C" int32_t ferrule_hip_kv_cache_append_launch(const FerruleHipKvCacheArgs *args) {
  return ferrule_hip::dispatch<ferrule_hip::Append>(args);
}
extern "C" int32_t ferrule_hip_kv_cache_read_can_implement(const FerruleHipKvCacheArgs *args) {
  return args == nullptr ? FERRULE_HIP_INVALID_ARGUMENT : ferrule_hip::validate_read(*args);
}
extern "C" int32_t ferrule_hip_kv_cache_read_launch(const FerruleHipKvCacheArgs *args) {
  return ferrule_hip::dispatch<ferrule_hip::Read>(args);
}
