// Attention over the MXFP4 key/value cache (no reference symbol; formats, layout and batch
// description: include/ferrule_hip_provider.h).
//
// Rows.  The n_b rows of a sequence times the `group` query heads of one key/value head are one list of packed
// rows r = row * group + head, cut into tiles: 16 rows are one column set of the matrix instructions, and one
// token for eight query heads fills half of it.
//
// One step takes 32 tokens through 16 rows, everything transposed so that a lane keeps ONE row from the scores to
// the output (lane = (i, g), i = lane % 16 the row, g = lane / 16):
//   S^T = K Q^T   v_mfma_scale_f32_16x16x128_f8f6f4: the cache's nibbles and scale bytes are the 4-bit operand as
//                 they stand; a BF16 row of q is split once into two E4M3 terms, x = q0 2^s0 + q1 2^s1
//                 (s1 = s0 - 5), exact but for elements below 2^-13 of their block's largest, which are held to
//                 2^-22 of it.
//   softmax       the two 16-token products are fed tokens 8(m/4) + m%4 and 4 more for their rows m, so lane
//                 (i, g) receives the scores of tokens 8g..8g+7 of row i: weights need no exchange between lanes
//                 before they are the next product's operand.
//   O^T += V^T P^T  v_mfma_f32_16x16x32_bf16: values cannot stay in 4 bits here (their scales run along the row,
//                 the sum runs over tokens), so they are expanded to BF16, exactly, and the weights are rounded
//                 to BF16: off by 2^-8 of a weight at most, as much as the output's own rounding, where 8-bit
//                 weights would be off by 2^-4; their sum is taken in f32 before that rounding.
// The running maximum of a row moves only when a score exceeds it by far (2^8 here, a lane's step of weights beyond
// 2^16 in the rows kernel; a wave-uniform branch): weights of that size cost a 32-bit sum nothing, and most steps
// rescale nothing.
//
// Two kernels, and two that join.  kv_attention_decode_kernel has 16 rows of which each wave takes its own tokens, four waves or
// eight, so that the cache is read once and in as many places as possible; its bound is memory.
// kv_attention_rows_kernel has 64 to 256 rows, its waves share the tokens and the expanded values; its bounds are
// the matrix pipe and, for heads of 64, the exponentials beside it.  Where rows leave CUs idle, the tokens of a
// tile are cut into parts of equal length for several workgroups, and (maximum, sum, O) of the parts are joined in
// a fixed order by the join kernels.
//   64 sequences of 8192 tokens, 8 heads of 128 for 8 query heads each: 102 us, 5.6 TB/s
//   the same with heads of 64: 59 us, 4.8 TB/s; 4096 tokens, heads of 256: 101 us, 5.6 TB/s
//   64 x 8192 tokens of one 512-wide row for 16 heads: 89 us, for 64 heads 124 us (the cache is 0.29 GB)
//   a prompt of 8192 tokens, 32 heads of 128: 470-480 us, 1.16 PFLOP/s (a large bf16 matrix product: 1.2)
//   heads of 64: 316 us, 0.87; 4096 tokens, 16 heads of 256: 145 us, 0.95; 1024 tokens, 64 of 512: 124 us, 0.55
// Here and below, unless a case of perf/operators.py is named (whose sequences are ragged): sequences of equal length on
// shuffled pages, between events over launches one after the other through the Python entry; "a, with .. b" is the same
// source with that one rule changed, "took a of what .. takes" a step's gain when it was made.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/ferrule_hip_provider.h"
#include "kv_cache.cuh"
#include "mx_core.cuh"

namespace ferrule_hip {
namespace {

constexpr uint32_t kWaves = 4;
constexpr uint32_t kTileRows = 16;   // packed rows of a tile
constexpr uint32_t kTileTokens = 32; // tokens of one step
constexpr float kLargest = 65536.0f; // rows kernel: sum of a lane's weights of one step that moves the maximum
constexpr float kLazy = 8.0f;        // how far (in powers of two) scores may exceed the running maximum

constexpr uint32_t kEveryRow = 0xffffffffu;

struct SplitPlan {
  uint32_t tile_rows;   // packed rows of a workgroup
  uint32_t page_shift;  // log2 of page_tokens
  uint32_t part_tiles;  // 32-token tiles of a part, at most unless there are `splits` of them
  uint32_t splits;      // parts at most
  uint32_t wide;        // decode kernel: workgroups of eight waves instead of parts, 1, or 2 with half of the values each
  uint32_t inner;       // decode kernel: tiles of rows are neighbours in the order of workgroups
  uint32_t find;        // rows kernel: workgroups are numbered by tile, not by sequence and tile
  uint32_t by_row;      // join: a workgroup for each of the rows there are, which looks for its sequence
  uint32_t least_rows;  // of the sequences that the launch is for
  uint32_t most_rows;   // kEveryRow: no bound
  uint32_t held_rows;   // rows for which a sequence has partials in the workspace, 0: they stand in the order of all rows
  uint64_t partials;    // byte offsets in the workspace
  uint64_t statistics;
};

// The 32-token tiles that a range of rows sees: tiles [0, head) and [first, first + count - head).
struct TileRange {
  uint32_t head;
  uint32_t first;
  uint32_t count;
  __device__ __forceinline__ uint32_t at(uint32_t v) const { return v < head ? v : first + (v - head); }
};

__device__ __forceinline__ TileRange tile_range(const FerruleHipKvAttentionArgs &a, int32_t low, int32_t high) {
  // rows at positions low..high; validate() keeps the table below 2^31 tokens
  TileRange t = {0u, 0u, 0u};
  const int32_t last = min(high, static_cast<int32_t>(a.max_pages * a.page_tokens) - 1);
  if (last < 0) return t;
  const uint32_t end = static_cast<uint32_t>(last) / kTileTokens + 1u;
  if (a.window != 0u) {
    const int32_t from = max(0, max(0, low) - static_cast<int32_t>(a.window - 1u));  // no row below 0 sees anything
    t.first = min(static_cast<uint32_t>(from) / kTileTokens, end);
    t.head = min((a.sinks + kTileTokens - 1u) / kTileTokens, t.first);
  }
  t.count = t.head + end - t.first;
  return t;
}

// A launch for the sequences of few rows leaves the others to its sibling, and the other way round.
__device__ __forceinline__ bool for_others(const KvSequence &s, const SplitPlan &plan) {
  return s.rows < plan.least_rows || s.rows > plan.most_rows;
}

// A tile of rows of some sequence.
struct RowTile {
  uint32_t b;
  uint32_t tile;
  bool there;
};

// Tile t of all that the sequences of the launch have, in their order, by the same rules as kv_sequence.  Workgroups
// without a tile would not only take time: workgroups go to the shader engines in turn, so their pattern decides which
// of those get the others (8 chunks of 200 to 600 rows in a grid for 600 each took 1.24 times what they take here, chunks of
// 2000, 100, 50 and 20 rows with the sequences faster than the tiles 2.5 times).
template <uint32_t ROWS>
__device__ __forceinline__ RowTile find_tile(const FerruleHipKvAttentionArgs &a, const SplitPlan &plan, uint32_t t, uint32_t lane,
                                             bool report) {
  const int32_t *indptr = global_ptr<const int32_t>(a.query_indptr), *lengths = global_ptr<const int32_t>(a.sequence_lengths);
  RowTile r = {0u, 0u, false};
  for (uint32_t from = 0u; from < a.batch; from += 64u) {
    const uint32_t l = from + lane;
    uint32_t tiles = 0u;
    if (l < a.batch) {
      const KvSequence s = kv_sequence_of(indptr[l], indptr[l + 1u], lengths[l], a.rows, a.max_query_length);
      if (report && s.bad) kv_report(a.error);
      if (!for_others(s, plan)) tiles = (s.rows * (a.q_heads / a.kv_heads) + ROWS - 1u) / ROWS;
    }
    uint32_t end = tiles;
#pragma unroll
    for (uint32_t step = 1u; step < 64u; step *= 2u) {
      const uint32_t below = static_cast<uint32_t>(__shfl_up(static_cast<int>(end), step, 64));
      end += lane >= step ? below : 0u;
    }
    const uint64_t behind = __ballot(end > t);
    if (behind != 0u && !r.there) {
      const uint32_t at = static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(behind))) - 1u;
      r.b = from + at;
      r.tile = t - static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(end - tiles), static_cast<int>(at)));
      r.there = true;
      if (!report) break;
    }
    t -= r.there ? 0u : static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(end), 63));
  }
  return r;
}

// How many parts a range has.
__device__ __forceinline__ uint32_t parts_of(uint32_t count, const SplitPlan &plan) {
  return max(1u, min((count + plan.part_tiles - 1u) / plan.part_tiles, plan.splits));
}

// Part `split` of them, all as long as the others (the last may be shorter, or empty): a long one behind a short one at
// every other workgroup would leave half of the XCDs, which take workgroups in turn, with the long ones.
struct PartRange {
  uint32_t begin, end;
};
__device__ __forceinline__ PartRange part_of(uint32_t count, uint32_t parts, uint32_t split) {
  const uint32_t length = (count + parts - 1u) / parts;
  return PartRange{min(split * length, count), min((split + 1u) * length, count)};
}

template <uint32_t D>
struct Core {
  using Layout = KvLayout<D>;
  static constexpr uint32_t kChunks = Layout::kKeyChunks;       // 128-value pieces of a row
  static constexpr uint32_t kTerms = D == 64u ? 1u : 2u;        // products per piece: both terms of 64 values fill one
  static constexpr uint32_t kUnits = D / 64u;                   // 16-byte value loads of a lane per 32 tokens
  static constexpr uint32_t kColumns = D / 16u;                 // accumulators of a tile

  template <uint32_t N>  // of a row's 128-value pieces
  struct QueryOf {
    static constexpr bool kRegisters = true;
    i32x8_t term[N * kTerms];
    uint32_t scale[N * kTerms];
    __device__ __forceinline__ i32x8_t get(uint32_t t, uint32_t &s) const {
      s = scale[t];
      return term[t];
    }
  };
  using Query = QueryOf<kChunks>;
  // The same in LDS, for waves that share their rows: at D = 512 the terms would take 72 registers.
  struct SharedQuery {
    u32x4_t term[kChunks * kTerms][2][64];
    uint32_t scale[kChunks * kTerms][64];
  };
  struct SharedReader {
    static constexpr bool kRegisters = false;
    const SharedQuery &q;
    uint32_t lane;
    __device__ __forceinline__ i32x8_t get(uint32_t t, uint32_t &s) const {
      s = q.scale[t][lane];
      return make_b_fp8(q.term[t][0][lane], q.term[t][1][lane]);
    }
  };
  template <uint32_t N>
  struct KeysOf {
    u32x4_t payload[N][2];
    uint2 scale[N];
  };
  using Keys = KeysOf<kChunks>;

  // 16 values of a row, as BF16 pairs
  struct Pairs {
    uint32_t w[8];
  };
  template <bool F32>
  static __device__ __forceinline__ Pairs load16(uint64_t base, uint64_t at) {
    Pairs r;
    if constexpr (F32) {
      const f32x4_t *src = reinterpret_cast<const f32x4_t *>(global_ptr<const float>(base) + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4_t x = src[i];
        r.w[2 * i] = __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(x[0]), static_cast<__bf16>(x[1])});
        r.w[2 * i + 1] = __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(x[2]), static_cast<__bf16>(x[3])});
      }
    } else {
      const u32x4_t *src = reinterpret_cast<const u32x4_t *>(global_ptr<const uint16_t>(base) + at);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u32x4_t x = src[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) r.w[4 * i + e] = x[e];
      }
    }
    return r;
  }

  // Exponent field of the largest magnitude of a block of 32: the lane's 16 values and lane ^ 16's.
  static __device__ __forceinline__ uint32_t block_field(const Pairs &x) {
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    u16x2_t top = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, x.w[i] & 0x7fff7fffu));
    const uint32_t most = max(static_cast<uint32_t>(top[0]), static_cast<uint32_t>(top[1]));
    return max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16, 64))) >> 7;
  }

  // Both terms of 16 values whose block's largest magnitude has the exponent field `field`; the converters take
  // the scale with them.
  static __device__ __forceinline__ uint32_t split16(const Pairs &x, uint32_t field, u32x4_t &q0, u32x4_t &q1) {
    typedef short i16x2_t __attribute__((ext_vector_type(2)));
    // largest magnitude to [128, 256): below E4M3's 448; the remainder is at most 2^3 of this scale, 2^8 of the next
    const uint32_t byte = min(max(field, 13u), 254u) - 7u;
    const float scale0 = __uint_as_float(byte << 23), scale1 = __uint_as_float((byte - 5u) << 23);
    const bool finite = field < 255u;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t lo = x.w[2 * w], hi = x.w[2 * w + 1];
      i16x2_t a = {0, 0}, b = {0, 0};
      a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, __builtin_bit_cast(bf16x2_t, lo), scale0, false);
      a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, __builtin_bit_cast(bf16x2_t, hi), scale0, true);
      const uint32_t first = __builtin_bit_cast(uint32_t, a);
      const f32x2_t back0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(first, scale0, false);
      const f32x2_t back1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(first, scale0, true);
      b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, __uint_as_float(lo << 16) - back0[0],
                                                   __uint_as_float(lo & 0xffff0000u) - back0[1], scale1, false);
      b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, __uint_as_float(hi << 16) - back1[0],
                                                   __uint_as_float(hi & 0xffff0000u) - back1[1], scale1, true);
      q0[w] = finite ? first : 0x7f7f7f7fu;  // a row with an infinity or a NaN: NaN scores
      q1[w] = finite ? __builtin_bit_cast(uint32_t, b) : 0u;
    }
    return byte;
  }

  // The lane's part of a 128-value piece of a tile's query rows, in two steps: what is asked for between
  // them need not wait for q.
  static constexpr uint32_t kHalves = D == 64u ? 1u : 2u;
  struct RawPiece {
    Pairs pairs[kHalves];
  };
  static __device__ __forceinline__ void load_query(uint64_t base, uint64_t row, uint32_t c, bool f32, uint32_t lane, RawPiece &raw) {
#pragma unroll
    for (uint32_t h = 0; h < kHalves; ++h) {
      const uint64_t at = row + c * 128u + h * 64u + (lane >> 4) * 16u;
      raw.pairs[h] = f32 ? load16<true>(base, at) : load16<false>(base, at);
    }
  }
  static __device__ __forceinline__ void split_query(const RawPiece &raw, uint32_t lane, i32x8_t (&term)[kTerms],
                                                     uint32_t (&scale)[kTerms]) {
    const uint32_t g = lane >> 4;
    const uint32_t source = (lane & 15u) + ((g & 1u) << 5);  // holds the scales of block g, in its half g / 2
    u32x4_t first[kHalves], second[kHalves];
    uint32_t byte[kHalves];
#pragma unroll
    for (uint32_t h = 0; h < kHalves; ++h) {
      const uint32_t own = split16(raw.pairs[h], block_field(raw.pairs[h]), first[h], second[h]);
      byte[h] = static_cast<uint32_t>(__shfl(static_cast<int>(own), static_cast<int>(source), 64));
    }
    if constexpr (D == 64u) {
      // values 0..63 twice along the product: first term against the first copy of a key, second against the second
      term[0] = make_b_fp8(first[0], second[0]);
      scale[0] = byte[0] - (g >= 2u ? 5u : 0u);
    } else {
      term[0] = make_b_fp8(first[0], first[kHalves - 1u]);
      term[kTerms - 1u] = make_b_fp8(second[0], second[kHalves - 1u]);
      scale[0] = g >= 2u ? byte[kHalves - 1u] : byte[0];
      scale[kTerms - 1u] = scale[0] - 5u;
    }
  }

  // Byte offsets of a lane's loads from the first byte of a 32-token tile (Place).
  struct Offsets {
    uint32_t key, key_scale, value, value_scale;
  };
  static __device__ __forceinline__ Offsets offsets(uint32_t lane) {
    const uint32_t i = lane & 15u, g = lane >> 4, block = D == 64u ? (g & 1u) : g;
    Offsets o;
    o.key = Layout::key_byte(8u * (i >> 2) + (i & 3u), 0u) + block * 16u;
    o.key_scale = Layout::key_scale(8u * (i >> 2), block);
    o.value = Layout::value_byte(8u * g, 2u * i);
    o.value_scale = Layout::value_scale(8u * g, i >> 3);
    return o;
  }

  // STREAM: read once, past the caches' other lines
  template <bool STREAM, typename T>
  static __device__ __forceinline__ T load(const uint8_t *p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const T *>(p));
    return *reinterpret_cast<const T *>(p);
  }

  template <bool STREAM, uint32_t N>  // pieces first .. first + N - 1
  static __device__ __forceinline__ void load_keys(const uint8_t *payload, const uint8_t *scales, const Offsets &o, KeysOf<N> &k,
                                                   uint32_t first = 0u) {
#pragma unroll
    for (uint32_t c = 0; c < N; ++c) {
#pragma unroll
      for (uint32_t half = 0; half < 2u; ++half) {
        k.payload[c][half] = load<STREAM, u32x4_t>(payload + o.key + ((first + c) * 32u + 4u * half) * Layout::kKeyBytes);
      }
      k.scale[c] = *reinterpret_cast<const uint2 *>(scales + o.key_scale + (first + c) * 128u);
    }
  }

  // One 16-byte piece of a lane: values 64u + 4i .. 64u + 4i + 3 of tokens 8g..8g+7, and their scale bytes.
  template <bool STREAM>
  static __device__ __forceinline__ void load_piece(const uint8_t *payload, const uint8_t *scales, uint32_t u, const Offsets &o,
                                                    u32x4_t &w, uint2 &scale) {
    w = load<STREAM, u32x4_t>(payload + o.value + u * 256u);
    scale = *reinterpret_cast<const uint2 *>(scales + o.value_scale + u * 16u);
  }

  // Scores of tokens 8g..8g+7 of row i: s[0..3] and s[4..7].
  template <uint32_t N, typename Q>
  static __device__ __forceinline__ void scores(const KeysOf<N> &k, const Q &q, uint32_t lane, f32x4_t (&s)[2]) {
    const uint32_t shift = 8u * (lane & 3u);
    s[0] = s[1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t c = 0; c < N; ++c) {
      const uint32_t scale[2] = {k.scale[c].x >> shift, k.scale[c].y >> shift};
#pragma unroll
      for (uint32_t term = 0; term < kTerms; ++term) {
        uint32_t q_scale;
        const i32x8_t q_term = q.get(c * kTerms + term, q_scale);
#pragma unroll
        for (uint32_t half = 0; half < 2u; ++half) {
          s[half] = mfma_fp4_fp8(make_a_fp4(k.payload[c][half]), q_term, s[half], scale[half], q_scale);
        }
      }
      // terms from LDS: not all of them at once, they would take the registers that the reader saves
      if constexpr (!Q::kRegisters) __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Blocks that cannot be multiplied: NaN (scale byte 255), and those whose largest values BF16 and f32 cannot hold
  // (4 * 2^126); both count as NaN.  The bytes' top bits, set for bytes of kLargestScale + 1 = 253 and more:
  static constexpr uint32_t kLargestScale = 252u;
  static __device__ __forceinline__ uint32_t not_finite(uint32_t scales) {
    return ((scales & 0x7f7f7f7fu) + 0x03030303u) & scales & 0x80808080u;
  }
  static __device__ __forceinline__ bool has_nan(const uint2 &scale) { return (not_finite(scale.x) | not_finite(scale.y)) != 0u; }
  static __device__ __forceinline__ uint2 without_nan(const uint2 &scale) {  // such bytes lose their top bit: 2^-2 .. 2^0
    return make_uint2(scale.x & ~not_finite(scale.x), scale.y & ~not_finite(scale.y));
  }

  // A block of NaN is expanded as if its scale were 1 or less, since 0 * NaN would reach rows that do not see it; the
  // rows that do take the NaN in the end.  Bit u: the lane's row sees a token whose values 16g .. 16g + 15 of the
  // 64 of unit first + u are NaN.  Rare, so it is kept small, and `scales` (of a 32-token tile) are read again.
  static __device__ __forceinline__ uint32_t nan_units(const uint8_t *scales, int32_t start, int32_t position, int32_t from,
                                                       int32_t sinks, uint32_t g, uint32_t first = 0u, uint32_t units_of = kUnits) {
    uint32_t units = 0u;
#pragma unroll 1
    for (uint32_t t = 0; t < kTileTokens; ++t) {
      const int32_t j = start + static_cast<int32_t>(t);
      const bool seen = j <= position && (j >= from || j < sinks);
#pragma unroll 1
      for (uint32_t u = 0; u < units_of; ++u) {
        const bool bad = scales[Layout::value_scale(t, 2u * (first + u) + (g >> 1))] > kLargestScale;
        units |= bad && seen ? 1u << u : 0u;
      }
    }
    return units;
  }

  // Four accumulators' operands from one 16-byte piece: values 64u + 4i + e of tokens 8g..8g+7, e = 0..3.
  static __device__ __forceinline__ void expand(const u32x4_t &w, const uint2 &scale, u32x4_t (&out)[4]) {
#pragma unroll
    for (uint32_t quad = 0; quad < 2u; ++quad) {  // four tokens
      const uint32_t bytes = quad == 0u ? scale.x : scale.y;
      const float s0 = __uint_as_float((bytes << 23) & 0x7f800000u), s1 = __uint_as_float((bytes << 15) & 0x7f800000u);
      const float s2 = __uint_as_float((bytes << 7) & 0x7f800000u), s3 = __uint_as_float((bytes >> 1) & 0x7f800000u);
#pragma unroll
      for (uint32_t pair = 0; pair < 2u; ++pair) {  // values 2 pair, 2 pair + 1
        const uint32_t x = w[2u * pair + quad];
        const uint32_t t0 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s0, 0));
        const uint32_t t1 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s1, 1));
        const uint32_t t2 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s2, 2));
        const uint32_t t3 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, s3, 3));
        out[2u * pair][2u * quad] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
        out[2u * pair][2u * quad + 1u] = __builtin_amdgcn_perm(t3, t2, 0x05040100u);
        out[2u * pair + 1u][2u * quad] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
        out[2u * pair + 1u][2u * quad + 1u] = __builtin_amdgcn_perm(t3, t2, 0x07060302u);
      }
    }
  }
};

// The largest (or the sum) of the four lanes that share a row.
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16, 64));
  return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float row_sum(float x) {
  x += __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

// What sums relative to the maximum `top` count for relative to `base`; sums that saw nothing (top
// -inf) are zeros, and an infinite weight would turn them to NaN.
__device__ __forceinline__ float part_weight(float top, float base) {
  return top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - base);
}

// Where a 32-token tile is.  An invalid one stands at page 0, so that what is loaded ahead for it is
// in bounds; nothing of it is used.
struct Place {
  uint32_t first;  // position of its first token
  uint64_t payload, scales;  // byte offsets
  bool valid;
};

// A tile's page comes from the table by a scalar load: page_of asks for it, place_at uses it, and a
// loop keeps a step or more between the two.  `count`: the range's tiles, at least 1.
__device__ __forceinline__ int32_t page_of(const FerruleHipKvAttentionArgs &a, const SplitPlan &plan, const TileRange &range,
                                           uint32_t b, uint32_t v, uint32_t count) {
  return kv_uniform(a.page_table,
                    static_cast<uint64_t>(b) * a.max_pages + ((range.at(min(v, count - 1u)) * kTileTokens) >> plan.page_shift));
}

template <uint32_t D>
__device__ __forceinline__ Place place_at(const FerruleHipKvAttentionArgs &a, const SplitPlan &plan, const TileRange &range,
                                          uint32_t kv_head, uint32_t v, uint32_t end, int32_t page, bool &bad) {
  Place p;
  p.first = range.at(v) * kTileTokens;
  p.valid = v < end && static_cast<uint32_t>(page) < a.page_count;
  bad |= v < end && !p.valid;
  // tokens in front of the tile, of every page and head
  const uint64_t head = static_cast<uint64_t>(p.valid ? static_cast<uint32_t>(page) : 0u) * a.kv_heads + kv_head;
  const uint64_t tokens = (head << plan.page_shift) + (p.valid ? p.first & (a.page_tokens - 1u) : 0u);
  p.payload = tokens * (D / 2u);
  p.scales = tokens * (D / 32u);
  return p;
}

// What a packed row is.  One behind the sequence's last stands at its first: what it computes is not written.
struct PackedRow {
  uint64_t q;       // offset of its values in q
  uint64_t output;  // and in the output
  uint64_t index;   // of its partials: row * q_heads + head
  int32_t position;
  bool live;
};

// Launches for sequences of few rows, and of fewer than the row tensors hold, have partials for those, held_rows to a
// sequence: of all rows' partials few would be used.
__device__ __forceinline__ PackedRow packed_row(const FerruleHipKvAttentionArgs &a, const SplitPlan &plan, const KvSequence &s,
                                                uint32_t b, uint32_t kv_head, uint32_t group, uint32_t r) {
  PackedRow p;
  const uint32_t row = r / group, head = kv_head * group + r % group;
  p.live = row < s.rows;
  const uint64_t at = s.row + static_cast<uint64_t>(p.live ? row : 0u);
  p.q = at * a.q_row_stride + head * a.q_head_stride;
  p.output = at * a.output_row_stride + head * a.output_head_stride;
  p.index = (plan.held_rows == 0u ? at : static_cast<uint64_t>(b) * plan.held_rows + row) * a.q_heads + head;
  p.position = s.position + static_cast<int32_t>(row);
  return p;
}

__device__ __forceinline__ uint32_t bf16_pair(float x, float y) {  // to nearest, ties to even
  return __builtin_bit_cast(uint32_t, bf16x2_t{static_cast<__bf16>(x), static_cast<__bf16>(y)});
}

// N consecutive values of a row
template <uint32_t N>
__device__ __forceinline__ void store(uint64_t output, uint64_t at, bool f32, const float (&x)[N]) {
  static_assert(N == 4u || N == 8u, "whole stores");
  if (f32) {
    float *dst = global_ptr<float>(output) + at;
#pragma unroll
    for (uint32_t q = 0; q < N / 4u; ++q) {
      reinterpret_cast<f32x4_t *>(dst)[q] = f32x4_t{x[4u * q], x[4u * q + 1u], x[4u * q + 2u], x[4u * q + 3u]};
    }
  } else {
    uint16_t *dst = global_ptr<uint16_t>(output) + at;
    uint32_t w[N / 2u];
#pragma unroll
    for (uint32_t e = 0; e < N / 2u; ++e) w[e] = bf16_pair(x[2u * e], x[2u * e + 1u]);
    if constexpr (N == 4u) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    if constexpr (N == 8u) *reinterpret_cast<u32x4_t *>(dst) = u32x4_t{w[0], w[1], w[2], w[3]};
  }
}

// Few rows: 16 of them, the token tiles shared out over the WAVES waves.  Keys and values go from memory to registers
// with loads that leave no line behind (decode of 64 x 8192 tokens, 8 heads of 128: with those and parts of equal length
// it took 0.85 of the time), a step ahead; what a wave has in flight, 4.25 KB at heads of 128, times 16 waves is 68 KB a CU.
// Heads of 256 and 512 have too many query terms for registers: one copy in LDS serves the four waves, and of a step's
// values four 16-byte pieces are in flight at a time (16 heads on a row of 512 took 0.64 of the time).
// At heads of 512 that leaves 244 registers and 136 accumulation registers a lane, one wave per SIMD: nothing runs while a
// step waits for its loads.
// Over a short range, eight waves, and two workgroups of them where there are CUs for it (COLUMNS = 2): both make the
// scores, each multiplies half of the values, whose expansion is half of a step's vector work.
// One sequence of 1000 tokens, 8 heads of 128 for 8 query heads each: 8.4 us (9.7 with one workgroup), of which 5 are a
// single step's chain of launch, table, cache and join; the others are a step's arithmetic, 0.7 us for two waves of a
// SIMD (loads two, three or four steps ahead change nothing).
template <uint32_t D>
constexpr uint32_t kDecodeOccupancy = D <= 128u ? 4u : D == 256u ? 2u : 1u;  // waves per SIMD that the registers allow
template <uint32_t D, uint32_t WAVES, uint32_t COLUMNS>
__global__ __launch_bounds__(WAVES * 64u, kDecodeOccupancy<D>) void kv_attention_decode_kernel(FerruleHipKvAttentionArgs a, SplitPlan plan) {
  using C = Core<D>;
  constexpr uint32_t kPitch = 128u + 4u;  // floats of a row in LDS
  constexpr bool kShared = D >= 256u;     // query terms in LDS
  constexpr uint32_t kUnits = C::kUnits / COLUMNS, kWidth = D / COLUMNS;  // of the values, the workgroup's
  constexpr uint32_t kRing = kUnits < 4u ? kUnits : 4u;
  __shared__ __align__(16) typename std::conditional<kShared, typename C::SharedQuery, uint32_t>::type shared;
  __shared__ __align__(16) float joined[WAVES][kTileRows][kPitch];
  __shared__ float top_of[WAVES][kTileRows], sum_of[WAVES][kTileRows];
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t i = lane & 15u, g = lane >> 4;
  const uint32_t b = blockIdx.y;
  const uint32_t split = blockIdx.x % plan.splits;
  const uint32_t kv_head = blockIdx.x / plan.splits % a.kv_heads;
  // 0 where COLUMNS is 1; taken from the grid there too at the sizes that have both (as a constant it costs heads of 128
  // three registers more, which spill: the case decode_batch 80 -> 86 us)
  const uint32_t outer = blockIdx.x / plan.splits / a.kv_heads;
  const uint32_t first_unit = (D == 128u || D == 256u) && plan.wide == 2u ? outer * kUnits : 0u;
  // the tile of rows is last in the order of workgroups: those that a sequence does not have are at the end, in nobody's
  // way (63 sequences of one row and one of four, 8192 tokens each, 8 heads, took 0.7 of the time).  Where every sequence
  // has all of them, they are neighbours, which share keys and values while those are in the cache (16 x 4 rows over 8192
  // tokens, 8 x 8 heads: 53 us, the other order 59; over a short range it costs 8 %).
  const uint32_t row_tile = plan.inner != 0u ? outer : blockIdx.z;
  const uint32_t group = a.q_heads / a.kv_heads;
  const KvSequence s = kv_sequence(a.query_indptr, a.sequence_lengths, b, a.rows, a.max_query_length);
  if (s.bad && blockIdx.x == 0u && blockIdx.z == 0u && threadIdx.x == 0u) kv_report(a.error);
  const uint32_t first_row = row_tile * kTileRows;
  if (first_row >= s.rows * group || for_others(s, plan)) return;
  const uint32_t last_row = min(first_row + kTileRows, s.rows * group) - 1u;
  const int32_t low = s.position + static_cast<int32_t>(first_row / group);
  const int32_t high = s.position + static_cast<int32_t>(last_row / group);
  const TileRange range = tile_range(a, low, high);
  if (high >= static_cast<int32_t>(a.max_pages * a.page_tokens) && threadIdx.x == 0u) kv_report(a.error);
  const uint32_t parts = parts_of(range.count, plan);
  if (split >= parts) return;
  const PartRange part = part_of(range.count, parts, split);
  const uint32_t begin = part.begin, end = part.end;
  const bool whole = parts == 1u;  // no join

  const PackedRow mine = packed_row(a, plan, s, b, kv_head, group, first_row + i);
  // a short range is a chain of memory latencies: the page number, then everything else at once
  bool bad = false;  // a page number outside the cache
  int32_t next_page = 0;
  Place next_place = {0u, 0u, 0u, false};
  const int32_t first_page = begin < end ? page_of(a, plan, range, b, begin + wave, end) : 0;
  if (begin < end) next_page = page_of(a, plan, range, b, begin + wave + WAVES, end);
  const bool f32_query = (a.flags & FERRULE_HIP_KV_ATTENTION_QUERY_F32) != 0u;
  typename C::RawPiece raw_query;  // the wave's piece: of few, every wave makes all, of several each makes one
  const uint32_t own_piece = kShared ? wave % C::kChunks : 0u;
  C::load_query(a.q, mine.q, own_piece, f32_query, lane, raw_query);
  if (begin < end) next_place = place_at<D>(a, plan, range, kv_head, begin + wave, end, first_page, bad);
  const uint8_t *k_payload = global_ptr<const uint8_t>(a.k_payload), *k_scales = global_ptr<const uint8_t>(a.k_scales);
  const uint8_t *v_payload = global_ptr<const uint8_t>(a.v_payload), *v_scales = global_ptr<const uint8_t>(a.v_scales);
  const typename C::Offsets offset = C::offsets(lane);
  typename C::Keys keys;
  // values: kRing 16-byte pieces, each taking the one kRing pieces on as soon as it is expanded
  u32x4_t ring[kRing];
  uint2 ring_scale[kRing];
  auto load_ring = [&](const Place &p) {
#pragma unroll
    for (uint32_t u = 0; u < kRing; ++u) {
      C::template load_piece<true>(v_payload + p.payload, v_scales + p.scales, first_unit + u, offset, ring[u], ring_scale[u]);
    }
  };
  C::template load_keys<true>(k_payload + next_place.payload, k_scales + next_place.scales, offset, keys);
  load_ring(next_place);
  i32x8_t term[C::kTerms];
  uint32_t term_scale[C::kTerms];
  C::split_query(raw_query, lane, term, term_scale);
  if constexpr (kShared) {
    if (wave < C::kChunks) {
#pragma unroll
      for (uint32_t t = 0; t < C::kTerms; ++t) {
        const uint32_t at = own_piece * C::kTerms + t;
        const u32x4_t lo = {static_cast<uint32_t>(term[t][0]), static_cast<uint32_t>(term[t][1]),
                            static_cast<uint32_t>(term[t][2]), static_cast<uint32_t>(term[t][3])};
        const u32x4_t hi = {static_cast<uint32_t>(term[t][4]), static_cast<uint32_t>(term[t][5]),
                            static_cast<uint32_t>(term[t][6]), static_cast<uint32_t>(term[t][7])};
        shared.term[at][0][lane] = lo;
        shared.term[at][1][lane] = hi;
        shared.scale[at][lane] = term_scale[t];
      }
    }
    lds_barrier();
  }
  typename C::Query own_query;
  if constexpr (!kShared) {
#pragma unroll
    for (uint32_t t = 0; t < C::kTerms; ++t) {
      own_query.term[t] = term[t];
      own_query.scale[t] = term_scale[t];
    }
  }
  const int32_t from = a.window == 0u ? static_cast<int32_t>(0x80000000u) : mine.position - static_cast<int32_t>(a.window - 1u);
  const int32_t sinks = a.window == 0u ? 0 : static_cast<int32_t>(a.sinks);
  const float factor = a.softmax_scale * 1.44269504088896341f;

  constexpr uint32_t kColumns = kWidth / 16u;
  f32x4_t out[kColumns];
#pragma unroll
  for (uint32_t c = 0; c < kColumns; ++c) out[c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  float top = -INFINITY, base = 0.0f, sum = 0.0f;  // base = top, or 0 while the row has seen nothing
  uint32_t nan_units = 0u;

  for (uint32_t v = begin + wave; v < end; v += WAVES) {
    // keys and values are loaded one step ahead, as soon as the registers of this step's are free; two or
    // three steps ahead at 3 or 2 waves per SIMD took 0.98 and 1.09 of the time (64 x 8192 tokens, 8 heads of 128)
    const Place here = next_place;
    next_place = place_at<D>(a, plan, range, kv_head, v + WAVES, end, next_page, bad);
    next_page = page_of(a, plan, range, b, v + 2u * WAVES, end);
    f32x4_t score[2];
    if constexpr (kShared) {
      C::scores(keys, typename C::SharedReader{shared, lane}, lane, score);
    } else {
      C::scores(keys, own_query, lane, score);
    }
    C::template load_keys<true>(k_payload + next_place.payload, k_scales + next_place.scales, offset, keys);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = score[e >> 2][e & 3];
    // tokens that every row of the tile sees need no mask
    const int32_t start = static_cast<int32_t>(here.first);
    const bool all = here.valid && start + 31 <= low && (a.window == 0u || start > high - static_cast<int32_t>(a.window) ||
                                                         start + 31 < static_cast<int32_t>(a.sinks));
    if (!all) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int32_t j = start + static_cast<int32_t>(8u * g) + e;
        x[e] = here.valid && j <= mine.position && (j >= from || j < sinks) ? x[e] : -INFINITY;
      }
    }
    float most = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7]))) * factor;
    if (__any(most > top + kLazy)) {
      most = fmaxf(top, row_max(most));
      const float next = most == -INFINITY ? 0.0f : most;
      const float keep = part_weight(top, next);  // 0 while nothing was seen: all sums are 0 then
      top = most;
      base = next;
      sum *= keep;
#pragma unroll
      for (uint32_t c = 0; c < kColumns; ++c) out[c] *= keep;
    }
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = __builtin_amdgcn_exp2f(fmaf(x[e], factor, -base));
    sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    bf16x8_t weight;
#pragma unroll
    for (int e = 0; e < 8; ++e) weight[e] = static_cast<__bf16>(w[e]);
    bool nan = false;
    if constexpr (kUnits <= 2u) {
#pragma unroll
      for (uint32_t u = 0; u < kUnits; ++u) nan |= C::has_nan(ring_scale[u]);
      if (__any(nan)) {
#pragma unroll
        for (uint32_t u = 0; u < kUnits; ++u) ring_scale[u] = C::without_nan(ring_scale[u]);
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < kUnits; ++u) {
      u32x4_t operand[4];
      if constexpr (kUnits <= 2u) {
        C::expand(ring[u], ring_scale[u], operand);
      } else {
        nan |= C::has_nan(ring_scale[u % kRing]);
        C::expand(ring[u % kRing], C::without_nan(ring_scale[u % kRing]), operand);
      }
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e) {
        out[4u * u + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, operand[e]), weight, out[4u * u + e], 0, 0, 0);
      }
      if constexpr (kUnits > 2u) {
        __builtin_amdgcn_sched_barrier(0);  // one piece's operands at a time
        const Place &source = u + kRing < kUnits ? here : next_place;
        C::template load_piece<true>(v_payload + source.payload, v_scales + source.scales, first_unit + (u + kRing) % kUnits, offset,
                                     ring[u % kRing], ring_scale[u % kRing]);
      }
    }
    if constexpr (kUnits <= 2u) load_ring(next_place);
    const bool nan_blocks = __any(nan);
    if (nan_blocks && here.valid) nan_units |= C::nan_units(v_scales + here.scales, start, mine.position, from, sinks, g, first_unit, kUnits);
  }

  if ((bad || low < 0) && lane == 0u) kv_report(a.error);  // rows in front of position 0 too
  // join the waves, 128 values at a time: 16 rows in pieces of kPiece
  constexpr uint32_t kPiece = 32u / WAVES, kPieces = 128u / kPiece;
  sum = row_sum(sum);
  if (g == 0u) {
    top_of[wave][i] = top;
    sum_of[wave][i] = sum;
  }
  __syncthreads();
  const uint32_t row_out = threadIdx.x / kPieces, d_out = threadIdx.x % kPieces * kPiece;
  float row_top = -INFINITY, total = 0.0f;
#pragma unroll
  for (uint32_t w = 0; w < WAVES; ++w) row_top = fmaxf(row_top, top_of[w][row_out]);
  const float row_base = row_top == -INFINITY ? 0.0f : row_top;
#pragma unroll
  for (uint32_t w = 0; w < WAVES; ++w) {
    total += sum_of[w][row_out] * part_weight(top_of[w][row_out], row_base);
  }
  float own_top = -INFINITY;
#pragma unroll
  for (uint32_t w = 0; w < WAVES; ++w) own_top = fmaxf(own_top, top_of[w][i]);
  const float keep = part_weight(top, own_top);
  const PackedRow target = packed_row(a, plan, s, b, kv_head, group, first_row + row_out);
  const bool seen_any = total != 0.0f;  // NaN too
  const float norm = whole ? (seen_any ? 1.0f / total : 0.0f) : 1.0f;
#pragma unroll
  for (uint32_t c = 0; c < (kWidth + 127u) / 128u; ++c) {
    if (c != 0u) __syncthreads();
#pragma unroll
    for (uint32_t u = 0; u < (kWidth < 128u ? 1u : 2u); ++u) {
#pragma unroll
      for (uint32_t e4 = 0; e4 < 4u; ++e4) {
        f32x4_t o;
#pragma unroll
        for (uint32_t e = 0; e < 4u; ++e) {
          o[e] = (nan_units >> (2u * c + u)) & 1u ? NAN : out[(2u * c + u) * 4u + e][e4] * keep;
        }
        *reinterpret_cast<f32x4_t *>(&joined[wave][i][64u * u + 16u * g + 4u * e4]) = o;
      }
    }
    __syncthreads();
    if (target.live && d_out < kWidth) {
      float x[kPiece] = {};
#pragma unroll
      for (uint32_t w = 0; w < WAVES; ++w) {
#pragma unroll
        for (uint32_t e = 0; e < kPiece; ++e) x[e] += joined[w][row_out][d_out + e];
      }
#pragma unroll
      for (uint32_t e = 0; e < kPiece; ++e) x[e] *= norm;
      const uint32_t d = first_unit * 64u + c * 128u + d_out;
      if (whole) {
        store<kPiece>(a.output, target.output + d, (a.flags & FERRULE_HIP_KV_ATTENTION_OUTPUT_F32) != 0u, x);
      } else {
        store<kPiece>(a.workspace + plan.partials, (target.index * plan.splits + split) * D + d, true, x);
      }
    }
  }
  if (!whole && target.live && threadIdx.x % kPieces == 0u) {
    global_ptr<float2>(a.workspace + plan.statistics)[target.index * plan.splits + split] = make_float2(row_top, total);
  }
}

// Many rows: 16 * NQ of them to a wave, and the WAVES waves of a workgroup go through the same tokens.
// Values are expanded to BF16 once per workgroup: a step has as many 16-byte pieces (D/64 per 32 tokens)
// as waves, or twice that, and every wave expands its own into the operands of four accumulators, in LDS,
// one step ahead of their use; keys are read by every wave, from cache, as they stand.  One barrier per step.
// Heads of 128 take 256 rows in eight waves: per 32 tokens and 16 rows the matrix pipe is busy for 256 cycles, the
// vector pipe for about 230 (8 exponentials of 16 cycles each, and their sums, conversions and address steps): 41 %
// and 50 % busy by the counters, at 2.1 GHz.  Heads of 64 halve the first and not the second: 32 % and 54 %.
// Eight waves have the next tile's scores made before this one's weights, so that neither waits for the other (heads of
// 256, 128 rows, chunks of 512 rows took 0.82 of the time; a prompt of 4096 tokens, heads of 128, 0.97; four waves gain
// nothing).  At heads of 512 a wave's accumulators alone are half of the registers, so that only four waves of 16 rows
// would stand on a CU, one for a SIMD: instead SHARES = 2 waves have the same 16 rows, each half of the values, and
// add up their halves of the scores in LDS (chunks of 512 rows for 64 heads took 0.77 of the time, four shares of 32 rows
// 0.86; 4 x 512 rows over 4096 tokens take 1330 us, 0.77 PFLOP/s).
// <128, 2, 8, 1> and <64, 4, 4, 1> keep 8 and 9 registers in scratch memory, stored in front of their loops and loaded
// behind them.
template <uint32_t D, uint32_t NQ, uint32_t WAVES, uint32_t SHARES>
struct Rows {
  static constexpr uint32_t kUnits = D / 64u;
  static constexpr uint32_t kShareUnits = kUnits / SHARES;  // of values and of the output, a wave's
  static constexpr uint32_t kShareChunks = Core<D>::kChunks / SHARES;  // of queries and keys
  static constexpr uint32_t kPieces = kUnits > WAVES ? kUnits : WAVES;  // of a step
  static constexpr uint32_t kOwn = kPieces / WAVES;                     // of them, a wave's
  static constexpr uint32_t kSub = kPieces / kUnits;                    // 32-token tiles of a step
  static constexpr bool kAhead = WAVES == 8u;  // the next tile's scores are made before this one's weights
  static constexpr uint32_t kInner = kAhead || NQ >= 4u || kSub < 2u ? 1u : 2u;  // tiles between two looks at the maximum
  static constexpr uint32_t kRows = 16u * NQ * WAVES / SHARES;
  static constexpr uint32_t kOccupancy = 2u;  // waves per SIMD: one workgroup of eight waves on a CU, or two of four
};

template <uint32_t D, uint32_t NQ, uint32_t WAVES, uint32_t SHARES>
__global__ __launch_bounds__(WAVES * 64u, (Rows<D, NQ, WAVES, SHARES>::kOccupancy)) void kv_attention_rows_kernel(
    FerruleHipKvAttentionArgs a, SplitPlan plan) {
  using C = Core<D>;
  using R = Rows<D, NQ, WAVES, SHARES>;
  constexpr uint32_t kSub = R::kSub, kInner = R::kInner, kOwn = R::kOwn;
  constexpr bool kAhead = R::kAhead;
  static_assert(SHARES == 1u || (kAhead && kSub == 1u), "shares of scores are exchanged once a step");
  __shared__ __align__(16) u32x4_t staged[2][R::kPieces][4][64];  // operands [piece][accumulator][lane]
  __shared__ uint32_t nan_of[2][WAVES];
  __shared__ __align__(16) f32x4_t shared_scores[2][SHARES > 1u ? WAVES : 1u][SHARES > 1u ? NQ * 2u : 1u][64];
  const uint32_t lane = threadIdx.x & 63u;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t i = lane & 15u, g = lane >> 4;
  const uint32_t share = wave % SHARES, first_unit = share * R::kShareUnits, first_chunk = share * R::kShareChunks;
  const uint32_t split = blockIdx.x % plan.splits;
  const uint32_t kv_head = blockIdx.x / plan.splits % a.kv_heads;
  const uint32_t group = a.q_heads / a.kv_heads;
  RowTile at = {blockIdx.y, blockIdx.x / plan.splits / a.kv_heads, true};
  if (plan.find != 0u) {
    at = find_tile<R::kRows>(a, plan, at.tile, lane, blockIdx.x == 0u && wave == 0u);
    if (!at.there) return;
  }
  const uint32_t b = __builtin_amdgcn_readfirstlane(at.b), row_tile = __builtin_amdgcn_readfirstlane(at.tile);
  const KvSequence s = kv_sequence(a.query_indptr, a.sequence_lengths, b, a.rows, a.max_query_length);
  if (plan.find == 0u && s.bad && blockIdx.x == 0u && threadIdx.x == 0u) kv_report(a.error);
  const uint32_t all_rows = s.rows * group;
  const uint32_t tiles = (all_rows + R::kRows - 1u) / R::kRows;
  if (row_tile >= tiles || for_others(s, plan)) return;
  const uint32_t first_row = (tiles - 1u - row_tile) * R::kRows;  // the longest causal ranges first
  const uint32_t last_row = min(first_row + R::kRows, all_rows) - 1u;
  const int32_t high = s.position + static_cast<int32_t>(last_row / group);
  const TileRange range = tile_range(a, s.position + static_cast<int32_t>(first_row / group), high);
  if (high >= static_cast<int32_t>(a.max_pages * a.page_tokens) && threadIdx.x == 0u) kv_report(a.error);
  const uint32_t parts = parts_of(range.count, plan);
  if (split >= parts) return;
  const PartRange part = part_of(range.count, parts, split);
  const uint32_t begin = part.begin, end = part.end;
  const bool whole = parts == 1u;

  // the wave's own rows
  const uint32_t wave_row = first_row + wave / SHARES * 16u * NQ;
  const int32_t wave_low = s.position + static_cast<int32_t>(min(wave_row, last_row) / group);
  const int32_t wave_high = s.position + static_cast<int32_t>(min(wave_row + 16u * NQ - 1u, last_row) / group);
  int32_t position[NQ], from[NQ];
  uint64_t row_q[NQ];
#pragma unroll
  for (uint32_t n = 0; n < NQ; ++n) {
    const PackedRow row = packed_row(a, plan, s, b, kv_head, group, wave_row + 16u * n + i);
    position[n] = row.position;
    from[n] = a.window == 0u ? static_cast<int32_t>(0x80000000u) : row.position - static_cast<int32_t>(a.window - 1u);
    row_q[n] = row.q;
  }
  const int32_t sinks = a.window == 0u ? 0 : static_cast<int32_t>(a.sinks);
  const float factor = a.softmax_scale * 1.44269504088896341f;
  constexpr uint32_t kColumns = C::kColumns / SHARES;
  f32x4_t out[NQ][kColumns];
  float top[NQ], base[NQ], sum[NQ];
  uint32_t nan_units[NQ];
  bool unset = true;  // some row has seen no token yet
#pragma unroll
  for (uint32_t n = 0; n < NQ; ++n) {
    top[n] = -INFINITY;
    base[n] = sum[n] = 0.0f;
    nan_units[n] = 0u;
#pragma unroll
    for (uint32_t c = 0; c < kColumns; ++c) out[n][c] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const uint8_t *k_payload = global_ptr<const uint8_t>(a.k_payload), *k_scales = global_ptr<const uint8_t>(a.k_scales);
  const uint8_t *v_payload = global_ptr<const uint8_t>(a.v_payload), *v_scales = global_ptr<const uint8_t>(a.v_scales);
  const typename C::Offsets offset = C::offsets(lane);
  bool bad = false;  // a page number outside the cache
  u32x4_t raw[kOwn];
  uint2 raw_scale[kOwn];
  bool raw_valid[kOwn];
  const uint32_t own_tile = wave * kOwn / C::kUnits;  // of a step: the tile that holds the wave's pieces
  auto load_pieces = [&](uint32_t v, int32_t page) {
    const Place p = place_at<D>(a, plan, range, kv_head, v + own_tile, end, page, bad);
#pragma unroll
    for (uint32_t o = 0; o < kOwn; ++o) {
      raw_valid[o] = p.valid;
      C::template load_piece<false>(v_payload + p.payload, v_scales + p.scales, (wave * kOwn + o) % C::kUnits, offset, raw[o],
                                    raw_scale[o]);
    }
  };
  auto stage_pieces = [&](uint32_t buffer) {
    bool nan = false;
#pragma unroll
    for (uint32_t o = 0; o < kOwn; ++o) {
      if (!raw_valid[o]) {  // of no use, but 0 * it has to be 0
        raw[o] = u32x4_t{0u, 0u, 0u, 0u};
        raw_scale[o] = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
      }
      nan |= C::has_nan(raw_scale[o]);
      u32x4_t operand[4];
      C::expand(raw[o], C::without_nan(raw_scale[o]), operand);
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e) staged[buffer][wave * kOwn + o][e][lane] = operand[e];
    }
    const uint32_t any = __any(nan) ? 1u : 0u;
    if (lane == 0u) nan_of[buffer][wave] = any;
  };
  typename C::template KeysOf<R::kShareChunks> keys[kInner];
  int32_t start[kInner];
  bool there[kInner];
  auto load_tiles = [&](uint32_t v, const int32_t *page) {
#pragma unroll
    for (uint32_t t = 0; t < kInner; ++t) {
      const Place p = place_at<D>(a, plan, range, kv_head, v + t, end, page[t], bad);
      start[t] = static_cast<int32_t>(p.first);
      there[t] = p.valid;
      C::template load_keys<false>(k_payload + p.payload, k_scales + p.scales, offset, keys[t], first_chunk);
    }
  };
  auto page = [&](uint32_t v) { return page_of(a, plan, range, b, v, end); };

  int32_t now[kSub], next[kSub], piece_page = 0;  // pages of this step's tiles, of the next one's, of the next piece
  uint32_t buffer = 0u;
  if (begin < end) {
#pragma unroll
    for (uint32_t t = 0; t < kSub; ++t) now[t] = page(begin + t + (kAhead ? 2u : 0u));
    load_pieces(begin, page(begin + own_tile));
    int32_t first_pages[kInner];
#pragma unroll
    for (uint32_t t = 0; t < kInner; ++t) first_pages[t] = page(begin + t);
    load_tiles(begin, first_pages);
  }
  typename C::template QueryOf<R::kShareChunks> query[NQ];
#pragma unroll
  for (uint32_t n = 0; n < NQ; ++n) {
    typename C::RawPiece piece[R::kShareChunks];
#pragma unroll
    for (uint32_t c = 0; c < R::kShareChunks; ++c) {
      C::load_query(a.q, row_q[n], first_chunk + c, (a.flags & FERRULE_HIP_KV_ATTENTION_QUERY_F32) != 0u, lane, piece[c]);
    }
#pragma unroll
    for (uint32_t c = 0; c < R::kShareChunks; ++c) {
      i32x8_t term[C::kTerms];
      uint32_t scale[C::kTerms];
      C::split_query(piece[c], lane, term, scale);
#pragma unroll
      for (uint32_t t = 0; t < C::kTerms; ++t) {
        query[n].term[c * C::kTerms + t] = term[t];
        query[n].scale[c * C::kTerms + t] = scale[t];
      }
    }
  }
  f32x4_t later[NQ][2];  // scores of the tile behind this one, or a share of them
  int32_t later_first = 0;
  bool later_valid = false;
  auto look_ahead = [&](uint32_t v, const int32_t *page, uint32_t buffer) {
    later_first = start[0];
    later_valid = there[0];
#pragma unroll
    for (uint32_t n = 0; n < NQ; ++n) C::scores(keys[0], query[n], lane, later[n]);
    load_tiles(v, page);
    if constexpr (SHARES > 1u) {
#pragma unroll
      for (uint32_t n = 0; n < NQ; ++n) {
#pragma unroll
        for (uint32_t half = 0; half < 2u; ++half) shared_scores[buffer][wave][n * 2u + half][lane] = later[n][half];
      }
    }
  };
  if (begin < end) {
    if constexpr (kAhead) {
      const int32_t second = page(begin + 1u);
      look_ahead(begin + 1u, &second, 0u);
    }
    stage_pieces(0u);
    load_pieces(begin + kSub, page(begin + kSub + own_tile));
    piece_page = page(begin + 2u * kSub + own_tile);
    lds_barrier();  // not a full one: it would wait for the loads in flight
  }
  // Which line of the instruction cache the loop starts in is worth up to 3 % (heads of 64, 4 x 512 rows over 8192 tokens:
  // 166 to 171 us): not to depend on what stands in front of it.
  asm volatile(".p2align 6");
  for (uint32_t v = begin; v < end; v += kSub, buffer ^= 1u) {
#pragma unroll
    for (uint32_t t = 0; t < kSub; ++t) next[t] = page(v + kSub + t + (kAhead ? 2u : 0u));
    const int32_t later_piece = page(v + 3u * kSub + own_tile);
#pragma unroll
    for (uint32_t inner = 0; inner < kSub; inner += kInner) {
      f32x4_t score[NQ][kInner][2];
      int32_t first[kInner];
      bool valid[kInner];
      if constexpr (kAhead) {
        first[0] = later_first;
        valid[0] = later_valid;
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n) {
#pragma unroll
          for (uint32_t half = 0; half < 2u; ++half) {
            if constexpr (SHARES > 1u) {  // every wave adds the shares in the same order: the same bits in all of them
              f32x4_t x = shared_scores[buffer][wave - share][n * 2u + half][lane];
#pragma unroll
              for (uint32_t other = 1; other < SHARES; ++other) x += shared_scores[buffer][wave - share + other][n * 2u + half][lane];
              score[n][0][half] = x;
            } else {
              score[n][0][half] = later[n][half];
            }
          }
        }
        look_ahead(v + inner + 2u, now + inner, buffer ^ 1u);
      } else {
#pragma unroll
        for (uint32_t t = 0; t < kInner; ++t) {
          first[t] = start[t];
          valid[t] = there[t];
#pragma unroll
          for (uint32_t n = 0; n < NQ; ++n) C::scores(keys[t], query[n], lane, score[n][t]);
        }
        load_tiles(v + inner + kInner, inner + kInner < kSub ? now + (inner + kInner) % kSub : next);
      }
      if (inner == 0u) {
        stage_pieces(buffer ^ 1u);
        load_pieces(v + 2u * kSub, piece_page);
      }
#pragma unroll
      for (uint32_t t = 0; t < kInner; ++t) {
        // tokens that every row of the wave sees need no mask
        const bool all = valid[t] && first[t] + 31 <= wave_low &&
                         (a.window == 0u || first[t] > wave_high - static_cast<int32_t>(a.window) ||
                          first[t] + 31 < static_cast<int32_t>(a.sinks));
        if (!all) {
#pragma unroll
          for (uint32_t n = 0; n < NQ; ++n) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int32_t j = first[t] + static_cast<int32_t>(8u * g) + e;
              const bool seen = valid[t] && j <= position[n] && (j >= from[n] || j < sinks);
              score[n][t][e >> 2][e & 3] = seen ? score[n][t][e >> 2][e & 3] : -INFINITY;
            }
          }
        }
      }
      // Weights relative to the maximum as it stands.  Whether that is too low shows in their sum, which is
      // needed anyway; only then (and until every row has seen a token) is the maximum looked for.
      bf16x8_t weight[NQ][kInner];
      float added[NQ];
      for (bool again = unset;; again = true) {
        if (again) {
          bool none = false;
#pragma unroll
          for (uint32_t n = 0; n < NQ; ++n) {
            float most = -INFINITY;
#pragma unroll
            for (uint32_t t = 0; t < kInner; ++t) {
#pragma unroll
              for (int e = 0; e < 8; ++e) most = fmaxf(most, score[n][t][e >> 2][e & 3]);
            }
            const float next_top = fmaxf(top[n], row_max(most) * factor);
            const float next_base = next_top == -INFINITY ? 0.0f : next_top;
            const float keep = part_weight(top[n], next_base);
            top[n] = next_top;
            base[n] = next_base;
            sum[n] *= keep;
#pragma unroll
            for (uint32_t c = 0; c < kColumns; ++c) out[n][c] *= keep;
            none |= next_top == -INFINITY;
          }
          unset = __any(none);
        }
        bool grows = false;
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n) {
          added[n] = 0.0f;
#pragma unroll
          for (uint32_t t = 0; t < kInner; ++t) {
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              w[e] = __builtin_amdgcn_exp2f(fmaf(score[n][t][e >> 2][e & 3], factor, -base[n]));
              weight[n][t][e] = static_cast<__bf16>(w[e]);
            }
            added[n] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
          }
          grows |= added[n] > kLargest;
        }
        if (again || !__any(grows)) break;
      }
#pragma unroll
      for (uint32_t n = 0; n < NQ; ++n) sum[n] += added[n];
      // the value operands come from LDS kRing products ahead
      constexpr uint32_t kOperands = kInner * kColumns, kRing = kOperands < 8u ? kOperands : SHARES > 1u ? 4u : 8u;
      u32x4_t ring[kRing];
      const u32x4_t(*operands)[64] = staged[buffer][inner * C::kUnits + first_unit];  // the share's of a tile; the next tile's
      constexpr uint32_t kTileOperands = C::kUnits * 4u;                              // are this far on
#pragma unroll
      for (uint32_t f = 0; f < kRing; ++f) ring[f] = operands[f / kColumns * kTileOperands + f % kColumns][lane];
#pragma unroll
      for (uint32_t f = 0; f < kOperands; ++f) {
        const uint32_t t = f / kColumns, c = f % kColumns, ahead = f + kRing;
        const bf16x8_t operand = __builtin_bit_cast(bf16x8_t, ring[f % kRing]);
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n) {
          out[n][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand, weight[n][t], out[n][c], 0, 0, 0);
        }
        if (ahead < kOperands) ring[f % kRing] = operands[ahead / kColumns * kTileOperands + ahead % kColumns][lane];
      }
      __builtin_amdgcn_sched_group_barrier(0x100, kRing, 0);
#pragma unroll
      for (uint32_t f = 0; f < kOperands; ++f) {
        __builtin_amdgcn_sched_group_barrier(0x008, NQ, 0);
        if (f + kRing < kOperands) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
    }
#pragma unroll
    for (uint32_t t = 0; t < kSub; ++t) now[t] = next[t];
    piece_page = later_piece;
    uint32_t nan_blocks = 0u;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) nan_blocks |= nan_of[buffer][w];
    if (nan_blocks != 0u) {
#pragma unroll 1
      for (uint32_t t = 0; t < kSub; ++t) {
        const Place p = place_at<D>(a, plan, range, kv_head, v + t, end, page(v + t), bad);
        if (!p.valid) continue;
#pragma unroll
        for (uint32_t n = 0; n < NQ; ++n) {
          nan_units[n] |= C::nan_units(v_scales + p.scales, static_cast<int32_t>(p.first), position[n], from[n], sinks, g, first_unit, R::kShareUnits);
        }
      }
    }
    lds_barrier();
  }
  if ((bad || wave_low < 0) && lane == 0u) kv_report(a.error);  // rows in front of position 0 too

#pragma unroll
  for (uint32_t n = 0; n < NQ; ++n) {
    const PackedRow row = packed_row(a, plan, s, b, kv_head, group, wave_row + 16u * n + i);
    const float total = row_sum(sum[n]);
    if (!row.live) continue;
    const float norm = whole ? (total != 0.0f ? 1.0f / total : 0.0f) : 1.0f;
#pragma unroll
    for (uint32_t u = 0; u < R::kShareUnits; ++u) {
#pragma unroll
      for (uint32_t half = 0; half < 2u; ++half) {  // values 64u + 16g + 8 half .. of the share's
        float x[8];
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e) {
          x[e] = (nan_units[n] >> u) & 1u ? NAN : out[n][4u * u + (e & 3u)][2u * half + (e >> 2)] * norm;
        }
        const uint32_t d = 64u * (first_unit + u) + 16u * g + 8u * half;
        if (whole) {
          store(a.output, row.output + d, (a.flags & FERRULE_HIP_KV_ATTENTION_OUTPUT_F32) != 0u, x);
        } else {
          store(a.workspace + plan.partials, (row.index * plan.splits + split) * D + d, true, x);
        }
      }
    }
    if (!whole && g == 0u && share == 0u) {
      global_ptr<float2>(a.workspace + plan.statistics)[row.index * plan.splits + split] = make_float2(top[n], total);
    }
  }
}

// The last sequence whose rows start at `row` or before it.
__device__ __forceinline__ uint32_t sequence_of(const FerruleHipKvAttentionArgs &a, uint32_t row) {
  uint32_t low = 0u, high = a.batch - 1u;
  while (low < high) {
    const uint32_t middle = (low + high + 1u) / 2u;
    if (global_ptr<const int32_t>(a.query_indptr)[middle] <= static_cast<int32_t>(row)) {
      low = middle;
    } else {
      high = middle - 1u;
    }
  }
  return low;
}

// The row and the number of parts of the threads that join one (row, query head); 0: written already.
struct Joined {
  PackedRow row;
  uint32_t parts;
};
__device__ __forceinline__ Joined joined_row(const FerruleHipKvAttentionArgs &a, const SplitPlan &plan, const KvSequence &s,
                                             uint32_t b, uint32_t item) {
  const uint32_t group = a.q_heads / a.kv_heads;
  const uint32_t kv_head = item % a.kv_heads, r = item / a.kv_heads;
  Joined j;
  j.parts = 0u;
  if (r < s.rows * group && !for_others(s, plan)) {
    const uint32_t first_row = r / plan.tile_rows * plan.tile_rows;
    const uint32_t last_row = min(first_row + plan.tile_rows, s.rows * group) - 1u;
    j.parts = parts_of(tile_range(a, s.position + static_cast<int32_t>(first_row / group),
                                  s.position + static_cast<int32_t>(last_row / group)).count, plan);
    if (j.parts == 1u) j.parts = 0u;
  }
  j.row = packed_row(a, plan, s, b, kv_head, group, j.parts != 0u ? r : 0u);
  return j;
}

// Joins the parts of every row, in their order.  Up to kFewParts parts: a thread has four values of a
// row and everything it reads is asked for at once, so the launch is two memory latencies long.
constexpr uint32_t kFewParts = 8;
template <uint32_t D>
__global__ __launch_bounds__(256) void kv_attention_join_few_kernel(FerruleHipKvAttentionArgs a, SplitPlan plan) {
  constexpr uint32_t kQuads = D / 4u;
  const uint32_t quad = threadIdx.x % kQuads;
  uint32_t item = (blockIdx.x * 256u + threadIdx.x) / kQuads;
  uint32_t b = blockIdx.y;
  KvSequence s;
  if (plan.by_row == 0u) {
    s = kv_sequence(a.query_indptr, a.sequence_lengths, b, a.rows, a.max_query_length);
  } else {  // a lane's own
    const uint32_t row = item / a.q_heads;
    b = sequence_of(a, row);
    const int32_t *indptr = global_ptr<const int32_t>(a.query_indptr), *lengths = global_ptr<const int32_t>(a.sequence_lengths);
    s = kv_sequence_of(indptr[b], indptr[b + 1u], lengths[b], a.rows, a.max_query_length);
    if (row < s.row) return;
    item -= s.row * a.q_heads;
  }
  const Joined j = joined_row(a, plan, s, b, item);
  if (j.parts == 0u) return;
  const float2 *statistics = global_ptr<const float2>(a.workspace + plan.statistics) + j.row.index * plan.splits;
  const f32x4_t *partials = reinterpret_cast<const f32x4_t *>(global_ptr<const float>(a.workspace + plan.partials)) +
                            j.row.index * plan.splits * kQuads + quad;
  float2 part[kFewParts];
  f32x4_t value[kFewParts];
#pragma unroll
  for (uint32_t p = 0; p < kFewParts; ++p) {
    const uint32_t at = min(p, j.parts - 1u);
    part[p] = statistics[at];
    value[p] = partials[at * kQuads];
  }
  float top = -INFINITY, total = 0.0f;
#pragma unroll
  for (uint32_t p = 0; p < kFewParts; ++p) top = fmaxf(top, part[p].x);  // the last part again does not change it
  const float base = top == -INFINITY ? 0.0f : top;
  f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (uint32_t p = 0; p < kFewParts; ++p) {
    if (p >= j.parts) break;
    const float weight = part_weight(part[p].x, base);
    total += part[p].y * weight;
    x += value[p] * weight;
  }
  const float norm = total != 0.0f ? 1.0f / total : 0.0f;
  const float y[4] = {x[0] * norm, x[1] * norm, x[2] * norm, x[3] * norm};
  store(a.output, j.row.output + 4u * quad, (a.flags & FERRULE_HIP_KV_ATTENTION_OUTPUT_F32) != 0u, y);
}

// More parts: a workgroup per (row, query head).  The maximum and the sum go over all parts at once; the
// values are added by 256 / (D / 4) threads per four values, each over a fixed set of parts, and those
// sums in turn.
template <uint32_t D>
__global__ __launch_bounds__(256) void kv_attention_join_kernel(FerruleHipKvAttentionArgs a, SplitPlan plan) {
  constexpr uint32_t kQuads = D / 4u, kLanes = 256u / kQuads;
  __shared__ float wave_top[kWaves], wave_sums[kWaves];
  __shared__ __align__(16) f32x4_t added[256];
  uint32_t b = blockIdx.y, item = blockIdx.x;
  if (plan.by_row != 0u) b = __builtin_amdgcn_readfirstlane(sequence_of(a, item / a.q_heads));
  const KvSequence s = kv_sequence(a.query_indptr, a.sequence_lengths, b, a.rows, a.max_query_length);
  if (plan.by_row != 0u) {
    if (item / a.q_heads < s.row) return;
    item -= s.row * a.q_heads;  // joined_row leaves out what is behind the sequence's last row
  }
  const Joined j = joined_row(a, plan, s, b, item);
  if (j.parts == 0u) return;
  const float2 *statistics = global_ptr<const float2>(a.workspace + plan.statistics) + j.row.index * plan.splits;
  const f32x4_t *partials = reinterpret_cast<const f32x4_t *>(global_ptr<const float>(a.workspace + plan.partials)) +
                            j.row.index * plan.splits * kQuads;
  const uint32_t wave = threadIdx.x >> 6;
  float top = -INFINITY;
  for (uint32_t p = threadIdx.x; p < j.parts; p += 256u) top = fmaxf(top, statistics[p].x);
  top = wave_max(top);
  if ((threadIdx.x & 63u) == 0u) wave_top[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
  const float base = top == -INFINITY ? 0.0f : top;
  float total = 0.0f;
  for (uint32_t p = threadIdx.x; p < j.parts; p += 256u) {
    const float2 part = statistics[p];
    total += part.y * part_weight(part.x, base);
  }
  total = wave_sum(total);
  if ((threadIdx.x & 63u) == 0u) wave_sums[wave] = total;
  const uint32_t quad = threadIdx.x % kQuads;
  f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (uint32_t p = threadIdx.x / kQuads; p < j.parts; p += kLanes) {
    x += partials[p * kQuads + quad] * part_weight(statistics[p].x, base);
  }
  added[threadIdx.x] = x;
  __syncthreads();
  if (threadIdx.x >= kQuads) return;
#pragma unroll
  for (uint32_t l = 1; l < kLanes; ++l) x += added[l * kQuads + threadIdx.x];
  total = (wave_sums[0] + wave_sums[1]) + (wave_sums[2] + wave_sums[3]);
  const float norm = total != 0.0f ? 1.0f / total : 0.0f;
  const float y[4] = {x[0] * norm, x[1] * norm, x[2] * norm, x[3] * norm};
  store(a.output, j.row.output + 4u * threadIdx.x, (a.flags & FERRULE_HIP_KV_ATTENTION_OUTPUT_F32) != 0u, y);
}

uint32_t row_bound(const FerruleHipKvAttentionArgs &a) { return a.max_query_length < a.rows ? a.max_query_length : a.rows; }

uint64_t packed_rows(const FerruleHipKvAttentionArgs &a) { return static_cast<uint64_t>(row_bound(a)) * (a.q_heads / a.kv_heads); }

uint32_t row_tiles(const FerruleHipKvAttentionArgs &a, uint32_t tile_rows) {
  return static_cast<uint32_t>((packed_rows(a) + tile_rows - 1u) / tile_rows);
}

// 32-token tiles that a workgroup of tile_rows packed rows can see, at most.
uint64_t token_tiles(const FerruleHipKvAttentionArgs &a, uint32_t tile_rows) {
  uint64_t tokens = a.max_sequence_length;
  if (a.window != 0u) {
    const uint64_t seen = static_cast<uint64_t>(a.window) + a.sinks + tile_rows + 2u * kTileTokens;
    tokens = tokens < seen ? tokens : seen;
  }
  return tokens / kTileTokens + 1u;
}

constexpr uint32_t kSegments = 256;   // CUs
constexpr uint32_t kShortRange = 64;  // tiles that eight waves take without parts

// Tiles of rows of one head, at most: the longest sequence's for every sequence, or what all rows make.
uint64_t found_tiles(const FerruleHipKvAttentionArgs &a, uint32_t tile_rows) {
  const uint64_t each = static_cast<uint64_t>(a.batch) * row_tiles(a, tile_rows);
  const uint64_t all = static_cast<uint64_t>(a.rows) * (a.q_heads / a.kv_heads) / tile_rows + a.batch;
  return each < all ? each : all;
}

uint64_t segments_of(const FerruleHipKvAttentionArgs &a, uint32_t tile_rows) { return found_tiles(a, tile_rows) * a.kv_heads; }

// Rows that are most of what they see: their ranges differ.
bool rows_of_prompts(const FerruleHipKvAttentionArgs &a) {
  return 2ull * a.max_query_length > kTileTokens * token_tiles(a, 64u);
}

// Packed rows that are the decode kernel's over any range.
uint32_t few_packed(const FerruleHipKvAttentionArgs &a) { return a.head_dim == 512u ? 16u : 32u; }

// Which kernel: packed rows of a workgroup of kv_attention_rows_kernel, 0 for kv_attention_decode_kernel.
// The latter reads and expands the range once for every 16 rows.  Two tiles of 16 are worth that everywhere but at heads
// of 512 (64 sequences of 4096 tokens, 32 query heads to each: 4 heads of 128 55 us, rows kernel 66, of 64 32 and 44, of
// 256 90 and 112; one of 512 79 and 66), four where every tile has a CU and a range is so short that it needs no parts
// (16 sequences, 4 heads, 64 rows over a window of 1024: the rows kernel took 1.6 times as long at heads of 64, twice as
// long at 256; at 512 over 128 tokens 1.15 times, but over 256 tokens 0.67).
uint32_t rows_of_workgroup(const FerruleHipKvAttentionArgs &a) {
  const uint64_t rows = packed_rows(a);
  const bool wide = a.head_dim == 512u;
  if (rows <= few_packed(a)) return 0u;
  if (rows <= 64u && segments_of(a, kTileRows) <= kSegments && token_tiles(a, kTileRows) <= (wide ? 2u * kWaves : kShortRange)) return 0u;
  if (rows <= 64u || a.head_dim == 512u) return 64u;
  // A workgroup of more rows reads and expands the tokens less often (a prompt of 8192 tokens, 32 heads of 128: 473 us
  // with 256 rows, 504 with 128, 600 with 64).  But the ranges of a prompt's rows differ, and cutting them costs more
  // than it gives: two workgroups for a CU even them out (2048 tokens: 64, 58 and 54 us; 512 tokens: 24 with 256, 15 with 64).
  // Nor are there enough steps in a short range to pay for the larger start (16 prompts of 256 tokens: 41 and 37).
  const uint64_t range = token_tiles(a, 64u);
  const uint64_t total = static_cast<uint64_t>(a.rows) * a.q_heads;
  // And few workgroups of few steps, whatever their tiles, leave most CUs idle (12 x 270 rows of one head over a window of
  // 574: heads of 64 29 us with 256 rows, 14 with 64; of 128 31 and 18).
  uint32_t tile = a.head_dim == 256u || rows <= 128u ? 128u : 256u;
  while (tile > 64u && (range < 16u || (rows_of_prompts(a) && total < 512u * tile) ||
                        segments_of(a, tile) * (range / 16u) < kSegments)) {
    tile /= 2u;
  }
  return tile;
}

// Parts of all ranges together.
// Decode: 1024, which the card holds at once up to heads of 128 (64 sequences of 8192 tokens, 8 heads of 128: 101 us, with
// 2048 parts 109, with 512 98).  At 256 it holds 512 of them and at 512 values 256, so that 1024 take two rounds and four:
// 512 parts are faster there (4096 tokens, 8 heads of 256: 100 and 92 us; 16 heads on a row of 512: 89 and 72; 64 heads
// the same).  Rows: no more than fill it once, one workgroup of eight waves or two of four to a CU, and parts long enough
// to pay for their f32 partials (4 x 512 rows over 8192 tokens: 8 x 4 heads of 128 227 us, with 512 parts 260; of 64
// 167 us, with 256 parts 200; 100 rows of 2 heads over 4000 tokens took 0.6 of what parts of 16 tiles and more took).
uint32_t target_parts(uint32_t head_dim, uint32_t tiles) {
  if (tiles == 0u) return 1024u;
  const bool eight_waves = head_dim == 512u || (head_dim == 256u && tiles == 128u) || (head_dim == 128u && tiles == 256u);
  return eight_waves ? 256u : 512u;
}
constexpr uint32_t kLeastPart = 8;  // tiles

// How the token ranges are cut: into parts of equal length, so that sequences of different lengths give
// workgroups of the same work.
SplitPlan plan_splits(const FerruleHipKvAttentionArgs &a, uint32_t tiles, uint64_t segments, uint32_t held_rows) {
  SplitPlan plan = {};
  plan.tile_rows = tiles == 0u ? kTileRows : tiles;
  plan.page_shift = static_cast<uint32_t>(__builtin_ctz(a.page_tokens));
  plan.most_rows = kEveryRow;
  plan.held_rows = held_rows;
  plan.find = tiles != 0u && a.batch > 1u && row_tiles(a, plan.tile_rows) > 1u;
  const uint64_t range = token_tiles(a, plan.tile_rows);
  const uint64_t target = target_parts(a.head_dim, tiles);
  const uint64_t least = tiles != 0u && rows_of_prompts(a) ? 2u * kLeastPart : kLeastPart;
  uint64_t part = (segments * range + target - 1u) / target;
  part = part < least ? least : part;
  if (tiles != 0u && 2u * range < 3u * part && range <= kShortRange) part = range;  // not for a little more than one part
  // A range of a few steps of eight waves is not worth a second launch while there are CUs for all segments (32
  // sequences of 8 heads of 256: 1000 tokens 15.4 us, in parts 24; 2000 tokens 26 and 33).  At 512 values eight waves
  // with all of the values each would have half of the registers that they need (1 sequence of 500 tokens: 1.7 times the
  // time); halves of the values, as at 128 and 256, are not built there.
  if (tiles == 0u && a.head_dim <= 256u && part < range && range <= kShortRange && segments <= kSegments) {
    plan.wide = a.head_dim > 64u && 2u * segments <= kSegments ? 2u : 1u;
    part = range;
  }
  plan.inner = tiles == 0u && range > kShortRange && row_tiles(a, kTileRows) > 1u &&
               a.rows == static_cast<uint64_t>(a.batch) * a.max_query_length;
  uint64_t splits = (range + part - 1u) / part;
  plan.part_tiles = static_cast<uint32_t>(part < 0x40000000u ? part : 0x40000000u);
  plan.splits = static_cast<uint32_t>(splits);
  if (plan.splits == 1u) return plan;
  // a workgroup for every row that a sequence might have takes time, also where there is none
  plan.by_row = static_cast<uint64_t>(a.batch) * row_bound(a) > 2ull * a.rows && static_cast<uint64_t>(a.rows) * a.q_heads <= 0x7fffffull;
  // segments times parts are fewer than twice `target`: far below 2^64 bytes
  const uint64_t held = held_rows == 0u ? a.rows : static_cast<uint64_t>(a.batch) * held_rows;
  plan.statistics = held * a.q_heads * plan.splits * a.head_dim * sizeof(float);
  return plan;
}

// One launch, or two.  A few rows over a long range need many workgroups for their range, and in a kernel for many rows
// they would keep one at work long after the others (63 sequences of a row and one of 512 rows, 8192 tokens each, 64
// heads: seven times what two launches take): where a batch can hold both, each launch takes its own sequences.
struct Plans {
  SplitPlan plan;
  bool both;
  SplitPlan few;
  FerruleHipKvAttentionArgs few_sizes;  // the arguments with the bound of the few rows
};

// Bytes of what the parts leave: their values, and two floats of statistics for head_dim of them.
uint64_t parts_size(const FerruleHipKvAttentionArgs &a, const SplitPlan &plan) {
  const uint64_t values = plan.statistics - plan.partials;
  return (values + values / a.head_dim * 2u + 255u) & ~255ull;
}

Plans plans_of(const FerruleHipKvAttentionArgs &a) {
  Plans p = {};
  const uint32_t tiles = rows_of_workgroup(a), tile_rows = tiles == 0u ? kTileRows : tiles, group = a.q_heads / a.kv_heads;
  uint64_t segments = segments_of(a, tile_rows);
  if (tiles != 0u && a.batch > 1u) {
    const uint32_t limit = few_packed(a) / group, few = limit == 0u ? 1u : limit;
    p.few_sizes = a;
    p.few_sizes.max_query_length = few;
    const uint32_t few_tiles = rows_of_workgroup(p.few_sizes);
    p.both = few_tiles < tiles && few < row_bound(a) && token_tiles(a, kTileRows) > kShortRange &&
             a.rows <= static_cast<uint64_t>(a.batch - 1u) * a.max_query_length + few;
    if (p.both) {
      // sized for one row each
      const uint32_t few_rows = few_tiles == 0u ? kTileRows : few_tiles;
      p.few = plan_splits(p.few_sizes, few_tiles, static_cast<uint64_t>(a.batch) * a.kv_heads * ((group + few_rows - 1u) / few_rows), few);
      p.few.most_rows = few;
      p.few.inner = 0u;  // the sequences of many rows have no tile in it, so not every sequence has all of them
      // as many sequences as it takes to have all rows
      const uint64_t sequences = (a.rows + a.max_query_length - 1ull) / a.max_query_length;
      segments = (static_cast<uint64_t>(a.rows) * group / tile_rows + sequences) * a.kv_heads;
    }
  }
  // row tensors may hold more rows than the sequences have
  p.plan = plan_splits(a, tiles, segments, static_cast<uint64_t>(a.batch) * row_bound(a) < a.rows ? row_bound(a) : 0u);
  if (p.both) {
    p.plan.least_rows = p.few.most_rows + 1u;
    const uint64_t behind = parts_size(a, p.plan);
    p.few.partials += behind;
    p.few.statistics += behind;
  }
  return p;
}

// What the block itself takes.
uint64_t workspace_size(const FerruleHipKvAttentionArgs &a) {
  const Plans p = plans_of(a);
  return parts_size(a, p.plan) + (p.both ? parts_size(a, p.few) : 0u);
}

// A launch of smaller bounds can take more: fewer rows are cut into more parts.  What a program asks for once at its
// largest bounds has to hold for all of them, so it is an upper bound that grows with each.
//
// With n tiles of rows to a key/value head a range has at most ceil(t / n) parts, t = ceil(target / kv_heads), and one
// where n >= t.  The largest n * ceil(t / n) of n = 1 .. most < t: an n of s parts is at most (t - 1) / (s - 1), so
// that n * s <= (t - 1) * s / (s - 1), which falls with s.
uint64_t most_parts(uint64_t most, uint64_t t) {
  if (t <= 1u || most == 0u) return 0u;
  if (most >= t) most = t - 1u;
  const uint64_t s = (t + most - 1u) / most, here = most * s, fewer = (t - 1u) * (s + 1u) / s;
  return here > fewer ? here : fewer;
}

// (row, query head)s times parts in a launch of any smaller bounds: up to `tiles` tiles of rows a head, each with `per`
// packed rows at most, `held` (row, query head)s in all, ranges of up to `range` tiles.
uint64_t most_partials(const FerruleHipKvAttentionArgs &a, uint32_t target, uint64_t tiles, uint64_t per, uint64_t held, uint64_t range) {
  const uint64_t t = (target + a.kv_heads - 1u) / a.kv_heads, splits = (range + kLeastPart - 1u) / kLeastPart;
  if (t <= 1u || splits <= 1u) return 0u;
  const uint64_t by_parts = a.kv_heads * per * most_parts(tiles, t);
  const uint64_t cut = a.kv_heads * per * (t - 1u), by_range = (held < cut ? held : cut) * splits;
  return by_parts < by_range ? by_parts : by_range;
}

uint64_t workspace_bound(const FerruleHipKvAttentionArgs &a) {
  const uint32_t group = a.q_heads / a.kv_heads, limit = few_packed(a) / group, few = limit == 0u ? 1u : limit;
  const uint64_t packed = packed_rows(a), all = static_cast<uint64_t>(a.batch) * row_bound(a), rows = all < a.rows ? all : a.rows;
  const bool both = a.batch > 1u && packed > few_packed(a) && few < row_bound(a) && token_tiles(a, kTileRows) > kShortRange;
  uint64_t most = 0u, beside = 0u;  // of the launch for all sequences, or for those of many rows; of the one for few rows beside that
  const uint32_t kinds[] = {kTileRows, 64u, 128u, 256u};
  for (const uint32_t tile : kinds) {
    // whether rows_of_workgroup has this tile for so many packed rows or fewer
    const auto reaches = [&](uint64_t count) {
      return tile == kTileRows || (tile == 64u && count > few_packed(a)) || (tile == 128u && count > 64u && a.head_dim < 512u) ||
             (tile == 256u && count > 128u && a.head_dim < 256u);
    };
    const uint32_t target = target_parts(a.head_dim, tile == kTileRows ? 0u : tile);
    if (reaches(packed)) {
      // beside a launch for few rows, tiles are counted by all rows
      const uint64_t tiles = tile == kTileRows ? found_tiles(a, tile) : rows * group / tile + a.batch;
      const uint64_t partials = most_partials(a, target, tiles, packed < tile ? packed : tile, rows * a.q_heads, token_tiles(a, tile));
      most = most > partials ? most : partials;
    }
    if (both && reaches(few * group)) {  // tiles are counted for one row of each sequence
      const uint64_t each = (group + tile - 1u) / tile, sequences = a.batch;
      const uint64_t partials = most_partials(a, target, sequences * each, (few * group + each - 1u) / each, sequences * few * a.q_heads,
                                              token_tiles(a, tile));
      beside = beside > partials ? beside : partials;
    }
  }
  const uint64_t bytes = (a.head_dim + 2u) * sizeof(float);
  return ((most * bytes + 255u) & ~255ull) + ((beside * bytes + 255u) & ~255ull);
}

dim3 grid_of(const FerruleHipKvAttentionArgs &a, const SplitPlan &plan) {
  const uint32_t tiles = row_tiles(a, plan.tile_rows), each = a.kv_heads * plan.splits;
  if (plan.find != 0u) return dim3(static_cast<uint32_t>(found_tiles(a, plan.tile_rows)) * each);
  if (plan.inner != 0u) return dim3(tiles * each, a.batch);
  if (plan.tile_rows == kTileRows) return dim3(plan.wide == 2u ? 2u * each : each, a.batch, tiles);
  return dim3(tiles * each, a.batch);  // one sequence or one tile
}

bool grid_fits(const FerruleHipKvAttentionArgs &a, const SplitPlan &plan) {
  const uint64_t tiles = plan.find != 0u ? found_tiles(a, plan.tile_rows) : row_tiles(a, plan.tile_rows);
  return tiles * a.kv_heads * plan.splits <= 0x7fffffull &&
         (plan.splits == 1u || static_cast<uint64_t>(row_bound(a)) * a.q_heads <= 0x7fffffull);
}

// Scalar fields; validate() looks at the rest.
FerruleHipStatus validate_shape(const FerruleHipKvAttentionArgs &a) {
  if (a.q_heads == 0u || a.kv_heads == 0u || a.q_heads % a.kv_heads != 0u || a.head_dim == 0u || a.page_count == 0u ||
      a.max_pages == 0u || a.max_query_length == 0u || !kv_page_tokens_valid(a.page_tokens) ||
      a.page_count > 0x7fffffffu || a.rows > 0x7fffffffu || a.window > 0x7fffffffu || a.sinks > 0x7fffffffu ||
      (a.flags & ~(FERRULE_HIP_KV_ATTENTION_QUERY_F32 | FERRULE_HIP_KV_ATTENTION_OUTPUT_F32)) != 0u ||
      !(a.softmax_scale > 0.0f && a.softmax_scale <= 0x1p127f)) {
    return FERRULE_HIP_INVALID_ARGUMENT;
  }
  if (!kv_head_dim_supported(a.head_dim)) return FERRULE_HIP_UNSUPPORTED;
  if (static_cast<uint64_t>(a.max_pages) * a.page_tokens > 0x7fffffffull) return FERRULE_HIP_UNSUPPORTED;
  // packed rows of a sequence count in 32 bits, and so do the threads of a grid's x (at most 512 to a workgroup)
  const uint64_t items = static_cast<uint64_t>(row_bound(a)) * a.q_heads;
  if (a.batch > 65535u || items > 0x0fffffffull) return FERRULE_HIP_UNSUPPORTED;
  const Plans p = plans_of(a);
  const bool fits = grid_fits(a, p.plan) && (!p.both || grid_fits(p.few_sizes, p.few));
  return fits ? FERRULE_HIP_SUCCESS : FERRULE_HIP_UNSUPPORTED;
}

FerruleHipStatus validate(const FerruleHipKvAttentionArgs &a) {
  if (a.batch == 0u || a.rows == 0u) return FERRULE_HIP_SUCCESS;  // nothing to do
  const FerruleHipStatus status = validate_shape(a);
  if (status == FERRULE_HIP_INVALID_ARGUMENT) return status;
  const uint32_t q_bytes = (a.flags & FERRULE_HIP_KV_ATTENTION_QUERY_F32) ? 4u : 2u;
  const uint32_t o_bytes = (a.flags & FERRULE_HIP_KV_ATTENTION_OUTPUT_F32) ? 4u : 2u;
  if (!kv_rows_aligned(a.q, a.rows, a.q_row_stride, a.q_heads, a.q_head_stride, q_bytes) ||
      !kv_rows_aligned(a.output, a.rows, a.output_row_stride, a.q_heads, a.output_head_stride, o_bytes) ||
      !kv_aligned16(a.k_payload) || !kv_aligned16(a.k_scales) || !kv_aligned16(a.v_payload) || !kv_aligned16(a.v_scales) || a.query_indptr == 0u ||
      a.sequence_lengths == 0u || a.page_table == 0u || ((a.query_indptr | a.sequence_lengths | a.page_table | a.error) & 3u)) {
    return FERRULE_HIP_INVALID_ARGUMENT;
  }
  // Two workgroups may read a query row of which each writes half of the output, and rows behind a sequence's last read
  // its first: the output is elsewhere.  What shows that it is not without a look at every row:
  if (a.q == a.output || (a.rows > 1u && a.output_row_stride == 0u) || (a.q_heads > 1u && a.output_head_stride == 0u)) {
    return FERRULE_HIP_INVALID_ARGUMENT;
  }
  if (status != FERRULE_HIP_SUCCESS) return status;
  const uint64_t needed = workspace_size(a);
  if (needed != 0u && (a.workspace == 0u || (a.workspace & 255u) != 0u || a.workspace_bytes < needed)) {
    return FERRULE_HIP_INVALID_ARGUMENT;
  }
  return FERRULE_HIP_SUCCESS;
}

template <uint32_t D>
void launch(const FerruleHipKvAttentionArgs &a, const FerruleHipKvAttentionArgs &sizes, const SplitPlan &plan, hipStream_t stream) {
  const dim3 grid = grid_of(sizes, plan);
  switch (rows_of_workgroup(sizes)) {
    case 0:
      if constexpr (D <= 256u) {
        if (plan.wide == 1u) {
          kv_attention_decode_kernel<D, 8, 1><<<grid, 512, 0, stream>>>(a, plan);
          break;
        }
      }
      if constexpr (D == 128u || D == 256u) {
        if (plan.wide == 2u) {
          kv_attention_decode_kernel<D, 8, 2><<<grid, 512, 0, stream>>>(a, plan);
          break;
        }
      }
      kv_attention_decode_kernel<D, kWaves, 1><<<grid, 256, 0, stream>>>(a, plan);
      break;
    case 64:
      if constexpr (D == 512u) kv_attention_rows_kernel<D, 1, 8, 2><<<grid, 512, 0, stream>>>(a, plan);
      if constexpr (D < 512u) kv_attention_rows_kernel<D, 1, 4, 1><<<grid, 256, 0, stream>>>(a, plan);
      break;
    case 128:
      if constexpr (D == 256u) kv_attention_rows_kernel<D, 1, 8, 1><<<grid, 512, 0, stream>>>(a, plan);
      if constexpr (D <= 128u) kv_attention_rows_kernel<D, 2, 4, 1><<<grid, 256, 0, stream>>>(a, plan);
      break;
    default:
      if constexpr (D == 64u) kv_attention_rows_kernel<D, 4, 4, 1><<<grid, 256, 0, stream>>>(a, plan);
      if constexpr (D == 128u) kv_attention_rows_kernel<D, 2, 8, 1><<<grid, 512, 0, stream>>>(a, plan);
      break;
  }
  if (plan.splits > 1u) {
    const uint32_t items = (plan.by_row != 0u ? a.rows : row_bound(sizes)) * a.q_heads, sequences = plan.by_row != 0u ? 1u : a.batch;
    if (plan.splits <= kFewParts) {
      constexpr uint32_t kRows = 256u / (D / 4u);
      kv_attention_join_few_kernel<D><<<dim3((items + kRows - 1u) / kRows, sequences), 256, 0, stream>>>(a, plan);
    } else {
      kv_attention_join_kernel<D><<<dim3(items, sequences), 256, 0, stream>>>(a, plan);
    }
  }
}

template <uint32_t D>
void launch(const FerruleHipKvAttentionArgs &a, hipStream_t stream) {
  const Plans p = plans_of(a);
  launch<D>(a, a, p.plan, stream);
  if (p.both) launch<D>(a, p.few_sizes, p.few, stream);
}

}  // namespace
}  // namespace ferrule_hip

extern "C" uint64_t ferrule_hip_kv_attention_workspace_size(const FerruleHipKvAttentionArgs *args) {
  using namespace ferrule_hip;
  if (args == nullptr || args->batch == 0u || args->rows == 0u || validate_shape(*args) != FERRULE_HIP_SUCCESS) return 0u;
  return workspace_bound(*args);
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
