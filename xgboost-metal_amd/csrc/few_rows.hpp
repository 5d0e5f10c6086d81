// Products with few rows (a request's, a single token's), out = x w^T: bound by the
// reading of w, once, and by the launch.
//
// A workgroup has 16 rows of w (result columns), its waves a share of the depth
// each, in units of one or four instructions (32 or 128 values), whose loads are all
// in flight; the waves' sums meet in LDS.  Where there are few such workgroups, the 16
// rows that an instruction takes of w are those of 8 columns in 2 slices of the depth,
// or of 4 in 4, and x's likewise: of its products those of equal slices count, and
// twice or four times as many workgroups read.
//
// Operands go from memory to registers in the matrix instruction's layout, whatever
// their alignment, and become bfloat16 or binary16 there: binary32 values three
// bfloat16 each (six instructions a product), blocks of 8 bits the values they stand
// for, exactly, and x, where the other operand is blocks, is rounded to blocks on the
// way (a block is a unit, and lies in the registers of four lanes).  Binary32 hidden
// values beside 16-bit matrices are two 16-bit values each.
#pragma once
#include "feed_forward.hpp"

namespace mgb {
namespace block {

// Above it tiles: 1,024 x 4,096 in bfloat16, 32 rows 18 us and 33, as tiles, 21 (64:
// 22); 256 x 1,024: 7 and 12.
constexpr int kMostFewRows = 32;

// Slices pay where workgroups are few.  1,024 x 4,096 in bfloat16, a row: 7.0 us, whole
// 11.8; 16 rows: 12.6, whole 15.2; 32 rows: 18.0, whole 20.3.  4,096 x 14,336, four rows:
// 96 us, whole 77.
constexpr int64_t kSlicedColumns = 4096, kSlicedDepth = 8192;

struct Few {
  const void* x;
  const void* w[2];              // the second for the dual form
  const uint8_t *x_scales, *w_scales[2];
  int64_t x_stride, w_stride[2];  // elements
  int64_t x_scale_stride, w_scale_stride;
  int64_t rows, columns, depth;
  void* out;                     // (rows, columns) without gaps
  float* kept;                   // (rows, 2, columns) or null
  int activation;
};

// How an operand lies: values of T; e4m3 blocks; x of T that is rounded to blocks.
template <typename T>
struct Plain {
  using Type = T;
  static constexpr int kParts = Kind<T>::kParts;
};
template <typename T>
struct Halves {  // binary32, each the sum of two of T
  using Type = float;
  using Half = T;
  static constexpr int kParts = 2;
};
struct InBlocks {
  using Type = uint8_t;
  static constexpr int kParts = 1;
};
template <typename T>
struct Rounded {
  using Type = T;
  static constexpr int kParts = 1;
};

// The exponent + 127 of the smallest power of two that takes `largest` to at most
// 448 = 1.75 2^8; 127 where there is none.
__device__ __forceinline__ uint32_t scale_of(float largest) {
  const uint32_t bits = __float_as_uint(largest);
  const int exponent = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return largest == 0.0f ? 127u : exponent > 0 ? (uint32_t)exponent : 0u;
}

__device__ __forceinline__ float scale_value(uint32_t scale) {  // 2^(scale - 127)
  return __uint_as_float(scale ? scale << 23 : 0x400000u);
}

// Eight values as e4m3, rounded to nearest even; infinities and NaN become its NaN.
__device__ __forceinline__ uint2 round_eight(const float* v, float factor) {
  int word[2] = {};
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    word[w] = __builtin_amdgcn_cvt_pk_fp8_f32(v[w * 4] * factor, v[w * 4 + 1] * factor, word[w], false);
    word[w] = __builtin_amdgcn_cvt_pk_fp8_f32(v[w * 4 + 2] * factor, v[w * 4 + 3] * factor, word[w], true);
  }
  return {(uint32_t)word[0], (uint32_t)word[1]};
}

// What eight e4m3 values times 2^(scale - 127) are, as bfloat16 (whose steps end at
// 2^-133); scale 255 is a block of NaN.
__device__ __forceinline__ product::bf16x8 widen_eight(uint2 bytes, uint32_t scale) {
  using Pair = __attribute__((ext_vector_type(2))) __bf16;
  const float factor = scale_value(scale);
  Pair v[4];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    v[w * 2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w ? bytes.y : bytes.x, factor, false);
    v[w * 2 + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w ? bytes.y : bytes.x, factor, true);
  }
  return __builtin_bit_cast(product::bf16x8, v);
}

// A unit of 16 rows: lane l has 8 values of row l % 16 for each of kSteps instructions.
template <class Kind_, int kSteps>
struct Unit {
  using T = typename Kind_::Type;
  static constexpr bool kBlocks = std::is_same_v<Kind_, InBlocks>;
  // 16 bytes a lane and load: 8 16-bit values, half of 8 binary32 ones, 16 of 8 bits.
  static constexpr int kLoads = kBlocks ? 2 : kSteps * (int)sizeof(T) / 2;
  static_assert(kSteps == 4 || !kBlocks, "a block is a unit");
  uint4 raw[kLoads];
  uint32_t scale;

  // Lane l / 16's 8 values of instruction s begin here; the same for both operands.
  static __device__ __forceinline__ int place(int s, int quarter, bool blocks) {
    return blocks ? s / 2 * 64 + quarter * 16 + s % 2 * 8 : s * 32 + quarter * 8;
  }
  // Rows beyond the last are read as zeros, as is the depth's end.
  __device__ __forceinline__ void load(const T* row, const uint8_t* scales, int64_t unit, int64_t depth, bool there,
                                       int quarter, bool with_blocks) {
    const int64_t begin = unit * (32 * kSteps);
    if constexpr (kBlocks) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        raw[k] = there ? *(const uint4*)(row + begin + k * 64 + quarter * 16) : uint4{};
      scale = there ? scales[unit] : 127u;
    } else {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int64_t at = begin + place(s, quarter, with_blocks);
        uint4 piece[sizeof(T) / 2] = {};
        if (there && at + 8 <= depth) {
          __builtin_memcpy(piece, row + at, sizeof(piece));
        } else if (there && at < depth) {
          T v[8] = {};
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (at + e < depth) v[e] = row[at + e];
          __builtin_memcpy(piece, v, sizeof(piece));
        }
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) raw[s * (sizeof(T) / 2) + k] = piece[k];
      }
    }
  }
  __device__ __forceinline__ void values(int s, float* v) const {
    T t[8];
    __builtin_memcpy(t, &raw[s * (sizeof(T) / 2)], sizeof(t));
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
  }
};

// x rounded to blocks: a unit's scale, of the four lanes that hold a row's.  Sizes are
// compared as integers, 16-bit ones two at once; infinities and NaN, the largest of
// them, are left out where there are any.
template <class Kind_, int kSteps>
__device__ __forceinline__ void find_scale(Unit<Kind_, kSteps>& u) {
  if constexpr (std::is_same_v<Kind_, Rounded<typename Kind_::Type>>) {
    using T = typename Kind_::Type;
    using Pair = __attribute__((ext_vector_type(2))) uint16_t;
    constexpr uint32_t kInfinite = sizeof(T) == 4 ? 0x7f800000u : std::is_same_v<T, _Float16> ? 0x7c00u : 0x7f80u;
    uint32_t most = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (const uint4& r : u.raw)
        most = max(max(most, max(r.x & 0x7fffffffu, r.y & 0x7fffffffu)), max(r.z & 0x7fffffffu, r.w & 0x7fffffffu));
    } else {
      Pair both = {};
#pragma unroll
      for (const uint4& r : u.raw)
#pragma unroll
        for (const uint32_t word : {r.x, r.y, r.z, r.w})
          both = __builtin_elementwise_max(both, __builtin_bit_cast(Pair, word & 0x7fff7fffu));
      most = max((uint32_t)both[0], (uint32_t)both[1]);
    }
    float largest;
    if (__any(most >= kInfinite)) {
      largest = 0.0f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        float v[8];
        u.values(s, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.0f);
      }
    } else if constexpr (sizeof(T) == 4) {
      largest = __uint_as_float(most);
    } else {
      largest = (float)__builtin_bit_cast(T, (uint16_t)most);
    }
    largest = fmaxf(largest, __shfl_xor(largest, 16, kWave));
    largest = fmaxf(largest, __shfl_xor(largest, 32, kWave));
    u.scale = scale_of(largest);
  }
}

// Instruction s's operand of a unit, in parts, from what was loaded.
template <class Kind_, int kSteps>
__device__ __forceinline__ void operand_of(const Unit<Kind_, kSteps>& u, int s, product::int4v* out) {
  if constexpr (std::is_same_v<Kind_, InBlocks>) {
    const uint2 bytes = s % 2 ? uint2{u.raw[s / 2].z, u.raw[s / 2].w} : uint2{u.raw[s / 2].x, u.raw[s / 2].y};
    out[0] = __builtin_bit_cast(product::int4v, widen_eight(bytes, u.scale));
  } else if constexpr (std::is_same_v<Kind_, Rounded<typename Kind_::Type>>) {
    float v[8];
    u.values(s, v);
    const uint2 bytes = round_eight(v, __uint_as_float((254u - u.scale) << 23));
    out[0] = __builtin_bit_cast(product::int4v, widen_eight(bytes, u.scale));
  } else if constexpr (Kind_::kParts == 2) {
    using Eight = __attribute__((ext_vector_type(8))) typename Kind_::Half;
    float v[8];
    u.values(s, v);
    Eight first, second;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      first[e] = (typename Kind_::Half)v[e];
      const float rest = v[e] - (float)first[e];
      second[e] = (typename Kind_::Half)(fabsf(rest) < INFINITY ? rest : 0.0f);
    }
    out[0] = __builtin_bit_cast(product::int4v, first);
    out[1] = __builtin_bit_cast(product::int4v, second);
  } else if constexpr (Kind_::kParts == 3) {
    float v[8];
    u.values(s, v);
    product::bf16x8 part[3];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      __bf16 three[3];
      split_parts(v[e], three);
#pragma unroll
      for (int q = 0; q < 3; ++q) part[q][e] = three[q];
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) out[q] = __builtin_bit_cast(product::int4v, part[q]);
  } else {
    out[0] = __builtin_bit_cast(product::int4v, u.raw[s]);
  }
}

template <bool kHalf>
__device__ __forceinline__ float4v multiply_one(product::int4v w, product::int4v x, float4v sum) {
  if constexpr (kHalf)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(product::f16x8, w), __builtin_bit_cast(product::f16x8, x),
                                                  sum, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(product::bf16x8, w),
                                                   __builtin_bit_cast(product::bf16x8, x), sum, 0, 0, 0);
}

// kTiles of 16 / kSlices rows of x; kDual: out = act(x w0^T) (x w1^T).
template <class X, class W, typename Out, int kTiles, int kSlices, bool kDual, int kWaves, int kSteps>
__global__ __launch_bounds__(kWaves* kWave) void k_few(Few p) {
  constexpr int kMatrices = kDual ? 2 : 1;
  constexpr bool kBlocks = std::is_same_v<W, InBlocks>;
  static_assert(X::kParts == W::kParts || (X::kParts == 2 && W::kParts == 1), "the products of parts that are made");
  constexpr int kColumns = 16 / kSlices, kRows = 16 / kSlices, kSums = 4 / kSlices;
  using Sum = __attribute__((ext_vector_type(kSums))) float;
  __shared__ Sum shared[kWaves][kMatrices][kTiles][kWave];
  using XT = typename X::Type;
  using WT = typename W::Type;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int quarter = lane / 16;
  const int slice = lane % kSlices;
  const int64_t column0 = (int64_t)blockIdx.x * kColumns, column = column0 + lane % 16 / kSlices;
  const bool column_there = column < p.columns;
  const WT* w[kMatrices];
  const uint8_t* w_scales[kMatrices];
#pragma unroll
  for (int m = 0; m < kMatrices; ++m) {
    w[m] = (const WT*)p.w[m] + (column_there ? column * p.w_stride[m] : 0);
    w_scales[m] = kBlocks ? p.w_scales[m] + (column_there ? column * p.w_scale_stride : 0) : nullptr;
  }
  const XT* x[kTiles];
  const uint8_t* x_scales[kTiles];
  bool row_there[kTiles];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    const int64_t row = t * kRows + lane % 16 / kSlices;
    row_there[t] = row < p.rows;
    x[t] = (const XT*)p.x + (row_there[t] ? row * p.x_stride : 0);
    x_scales[t] = std::is_same_v<X, InBlocks> ? p.x_scales + (row_there[t] ? row * p.x_scale_stride : 0) : nullptr;
  }
  float4v sum[kMatrices][kTiles] = {};
  const int64_t units = (p.depth + 32 * kSteps * kSlices - 1) / (32 * kSteps * kSlices);
  int64_t unit = units * wave / kWaves;
  const int64_t end = units * (wave + 1) / kWaves;
  Unit<W, kSteps> next_w[kMatrices];
  Unit<X, kSteps> next_x[kTiles];
  auto fetch = [&] {
    const int64_t at = unit * kSlices + slice;
    const bool within = kSlices == 1 || at * (32 * kSteps) < p.depth;
#pragma unroll
    for (int m = 0; m < kMatrices; ++m) next_w[m].load(w[m], w_scales[m], at, p.depth, column_there && within, quarter, kBlocks);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) next_x[t].load(x[t], x_scales[t], at, p.depth, row_there[t] && within, quarter, kBlocks);
  };
  // The next unit's loads are on their way while one is multiplied, where the
  // registers hold both.
  constexpr int kRaw = 4 * (kMatrices * Unit<W, kSteps>::kLoads + kTiles * Unit<X, kSteps>::kLoads);
  constexpr bool kAhead = 2 * kRaw <= (kWaves > 8 ? 64 : 192);
  if (kAhead && unit < end) fetch();
  while (unit < end) {
    if constexpr (!kAhead) fetch();
    Unit<W, kSteps> this_w[kMatrices];
    Unit<X, kSteps> this_x[kTiles];
#pragma unroll
    for (int m = 0; m < kMatrices; ++m) this_w[m] = next_w[m];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) this_x[t] = next_x[t];
    ++unit;
    if (kAhead && unit < end) fetch();
#pragma unroll
    for (int t = 0; t < kTiles; ++t) find_scale(this_x[t]);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      product::int4v of_w[kMatrices][W::kParts];
#pragma unroll
      for (int m = 0; m < kMatrices; ++m) operand_of(this_w[m], s, of_w[m]);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        product::int4v of_x[X::kParts];
        operand_of(this_x[t], s, of_x);
#pragma unroll
        for (int pair = 0; pair < (X::kParts == 3 ? Kind<float>::kPairs : X::kParts); ++pair) {
          const int xp = X::kParts == 3 ? product::left_part(pair) : pair, wp = X::kParts == 3 ? product::right_part(pair) : 0;
#pragma unroll
          for (int m = 0; m < kMatrices; ++m)
            sum[m][t] = multiply_one<std::is_same_v<W, Plain<_Float16>>>(of_w[m][wp], of_x[xp], sum[m][t]);
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kMatrices; ++m)
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int e = 0; e < kSums; ++e) shared[wave][m][t][lane][e] = group_sum<kSlices>(sum[m][t][e * kSlices + slice]);
  __syncthreads();
  auto finish = [&](int64_t row, int64_t column, float first, float second) {
    if (row >= p.rows || column >= p.columns) return;
    if constexpr (kDual) {
      if (p.kept) {
        p.kept[row * 2 * p.columns + column] = first;
        p.kept[(row * 2 + 1) * p.columns + column] = second;
      }
      first = activate<sizeof(Out) == 4>(first, p.activation) * second;
    }
    ((Out*)p.out)[row * p.columns + column] = (Out)first;
  };
  // A lane joins kSums columns of a row.
  for (int at = threadIdx.x; at < kTiles * kWave; at += kWaves * kWave) {
    const int t = at / kWave, l = at % kWave;
    Sum total[kMatrices];
#pragma unroll
    for (int m = 0; m < kMatrices; ++m) {
      total[m] = shared[0][m][t][l];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) total[m] += shared[k][m][t][l];
    }
    if (l % kSlices != 0) continue;
#pragma unroll
    for (int e = 0; e < kSums; ++e)
      finish(t * kRows + l % 16 / kSlices, column0 + l / 16 * kSums + e, total[0][e], total[kMatrices - 1][e]);
  }
}

template <class X, class W, typename Out, bool kDual>
void few_rows(const Few& p, hipStream_t stream) {
  // Waves for every unit, up to as many as the registers of their loads allow; units of
  // one instruction where there are fewer of four than waves.
  constexpr int kMost = kDual ? 8 : 16;
  constexpr bool kBlocks = std::is_same_v<W, InBlocks>;
  auto launch = [&](auto tiles, auto slices, auto waves, auto steps) {
    constexpr int kWaves = decltype(waves)::value, kSlices = decltype(slices)::value;
    const uint32_t groups = (uint32_t)((p.columns * kSlices + 15) / 16);
    k_few<X, W, Out, decltype(tiles)::value, kSlices, kDual, kWaves, decltype(steps)::value><<<groups, kWaves * kWave, 0, stream>>>(p);
  };
  auto with = [&](auto tiles, auto slices) {
    using One = std::integral_constant<int, 1>;
    using Four = std::integral_constant<int, 4>;
    using Most = std::integral_constant<int, (kBlocks && decltype(slices)::value > 1) ? 8 : kMost>;
    const int64_t depth = (p.depth + decltype(slices)::value - 1) / decltype(slices)::value;
    if constexpr (kBlocks) {
      if (depth > 512) launch(tiles, slices, Most{}, Four{});
      else launch(tiles, slices, Four{}, Four{});
    } else {
      if (depth <= 128) launch(tiles, slices, Four{}, One{});
      else if constexpr (sizeof(typename W::Type) == 4 || (sizeof(typename X::Type) == 4 && decltype(tiles)::value > 1))
        launch(tiles, slices, Most{}, One{});
      else if (depth < 128 * kMost) launch(tiles, slices, Most{}, One{});
      else launch(tiles, slices, Most{}, Four{});
    }
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  if (p.columns <= kSlicedColumns && p.depth <= kSlicedDepth) {
    if (p.rows <= 4) return with(One{}, Four{});
    if (p.rows <= 8) return with(One{}, Two{});
    if constexpr (!kBlocks)
      if (p.rows <= 16) return with(Two{}, Two{});
    if constexpr (!kBlocks && sizeof(typename W::Type) == 2) return with(Four{}, Two{});
  }
  if (p.rows <= 16) with(One{}, One{});
  else with(Two{}, One{});
}

}  // namespace block
}  // namespace mgb
