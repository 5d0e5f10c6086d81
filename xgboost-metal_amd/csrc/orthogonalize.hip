// A matrix's update made orthogonal by Newton-Schulz products (the Muon
// optimiser's update): with X0 = G / (|G|_F + eps), m x n and m <= n (taller
// ones transposed),
//   X <- (a I + b A + c A^2) X,   A = X X^T,   `steps` times.
// Every step is a polynomial Z in A applied from the left, so a segment of
// steps can run among m x m matrices: A <- Z A Z and P <- Z P, all symmetric and
// commuting, and one product X <- P X ends it.  For n > m that leaves out most
// products with n; symmetric results take half their tiles.  An error in A grows
// by a^2 a step where X is small, so a segment has at most three steps
// and the next one takes A from X anew (low rank 512 x 2048: 4e-5 of the norm with
// three, 2e-5 in plain binary32, 1e-4 with all five in one segment); with binary32
// results a segment is one step.
//
// The matrix instructions multiply binary16.  A small direction's part grows
// a-fold a step, so operands of 11 bits would show in the result (4e-2 of the
// norm at low rank, after five steps): each value is the sum of two binary16
// numbers, 22 bits, and a product takes three matrix instructions (high by
// high, high by low, low by high; low by low is below binary32's rounding).
// Sums are binary32.
//
// Measured (us, one MI355X, a call among others and from a graph): binary32 64 x 256 51
// and 1,500 x 1,001 252 and 224, bfloat16 2,048 x 4,096 943 and 881 (198 GFLOP, thrice in
// matrix instructions: 630 to 670 TFLOP/s of those, where a library's large product
// reaches 1,130).
#include <cmath>
#include <type_traits>
#include <utility>

#include "encoder_common.hpp"

namespace mgb {
namespace {

constexpr int kThreads = 256;
constexpr int kPad = 64;       // rows and columns of every matrix in the workspace are padded to whole 64s
constexpr int kNormGroups = 256;
constexpr int64_t kMostSide = int64_t(1) << 20;
constexpr float kMostCoefficient = 8.0f;
constexpr double kMostHalf = 65504.0 * 0.99;  // binary16's largest value, and room for roundings

// Steps of a segment at most: results of 24 bits show what a second step's error
// adds (512 x 2048: 3.5e-6 of the norm, 1.5e-6 with one, plain binary32 2.8e-6),
// those of 11 and 8 bits do not show a third's.
constexpr int kSegment32 = 1, kSegment16 = 3;

// What stored values are scaled by: X, A and U, whose entries may be up to 15.8 then
// (about 1 with coefficients that converge), and Z and P, up to 1,013 (a^kSegment16
// at most, which is 512).  in_range checks it.  A value of at least 2^-2 / scale keeps
// 22 bits; a smaller one is off by 2^-25 / scale.
constexpr float kScaleX = 4096.0f, kScaleZ = 64.0f;

using half8 = __attribute__((ext_vector_type(8))) _Float16;
using half4 = __attribute__((ext_vector_type(4))) _Float16;
using float4v = __attribute__((ext_vector_type(4))) float;
using float16v = __attribute__((ext_vector_type(16))) float;

// A matrix as the matrix instructions take it: blocks of 32 rows and 16 columns,
// the high parts' 1 KB before the low parts', where lane l's 16 bytes are row
// l % 32, columns l / 32 * 8 .. + 7.  A wave loads a block whole.
constexpr int kBlock = 32 * 16;
struct Split {
  _Float16* data;
  int64_t blocks;        // side by side: padded columns / 16
  int64_t batch_stride;  // elements
};

__device__ __forceinline__ _Float16* element(const Split& m, int64_t batch, uint32_t row, uint32_t column) {
  return m.data + batch * m.batch_stride + (row / 32 * m.blocks + column / 16) * (2 * kBlock) +
         (row % 32 + column % 16 / 8 * 32) * 8 + column % 8;
}

// Four values as high and low parts.
struct Parts {
  half4 high, low;
};

__device__ __forceinline__ Parts parts_of(float4v v) {
  Parts p;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    p.high[e] = (_Float16)v[e];
    p.low[e] = (_Float16)(v[e] - (float)p.high[e]);
  }
  return p;
}

// Where four that follow each other in a row go, from a column 4 k on.
__device__ __forceinline__ void store_parts(_Float16* to, const Parts& p) {
  *(half4*)to = p.high;
  *(half4*)(to + kBlock) = p.low;
}

__device__ __forceinline__ void store_four(_Float16* to, float4v v) { store_parts(to, parts_of(v)); }

// Lanes t = 0 .. 3 of a quad hold element [e][t] of a 4 x 4 as v[e]; afterwards
// [t][e]: pairs of lanes exchange halves of words, then pairs of pairs words.
__device__ __forceinline__ half4 turn_quads(half4 v) {
  uint32_t w[2];
  __builtin_memcpy(w, &v, sizeof(w));
  const bool odd = threadIdx.x & 1, upper = threadIdx.x & 2;
  const uint32_t halves = odd ? 0x03020706u : 0x05040100u;  // of (other, own): the upper ones, or the lower
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t other = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w[k], 0xb1, 0xf, 0xf, false);
    w[k] = __builtin_amdgcn_perm(other, w[k], halves);
  }
  const uint32_t got =
      (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(upper ? w[0] : w[1]), 0x4e, 0xf, 0xf, false);
  w[0] = upper ? got : w[0];
  w[1] = upper ? w[1] : got;
  __builtin_memcpy(&v, w, sizeof(w));
  return v;
}

__device__ __forceinline__ Parts turn_quads(const Parts& p) { return {turn_quads(p.high), turn_quads(p.low)}; }

__device__ __forceinline__ float4v load_four(const _Float16* from) {
  const half4 high = *(const half4*)from, low = *(const half4*)(from + kBlock);
  float4v v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)high[e] + (float)low[e];
  return v;
}

// A 32 x 32 of a product in registers: a lane's q-th four values are rows
// 8 q + 4 (lane / 32) .. + 3 of column lane % 32.  As it lies there it is four of a
// row of the transpose, row lane % 32; after an exchange among quads of lanes
// (turn_quads) four of row 8 q + 4 (lane / 32) + lane % 4 from column
// lane % 32 / 4 * 4 on.  The two places in a 32 x 32 in memory, from its first
// block on:
__device__ __forceinline__ int turned_place(int lane, int q) {
  return lane % 32 * 8 + lane / 32 * 4 + q / 2 * (2 * kBlock) + q % 2 * 256;
}
__device__ __forceinline__ int straight_place(int lane, int q) {
  return lane % 32 / 16 * (2 * kBlock) + (lane / 32 * 4 + lane % 4) * 8 + lane % 16 / 8 * 256 + lane % 8 / 4 * 4 + q * 64;
}
__device__ __forceinline__ _Float16* tile_of(const Split& m, int64_t batch, uint32_t row_tile, uint32_t column_tile) {
  return m.data + batch * m.batch_stride + ((int64_t)row_tile * m.blocks + 2 * column_tile) * (2 * kBlock);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_square_sums(float* __restrict__ partial, const T* __restrict__ g,
                                                          int64_t rows, int64_t columns, int64_t stride,
                                                          int64_t batch_stride) {
  __shared__ float shared[kThreads / kWave];
  constexpr int kSize = Pack<T>::kSize, kOnce = 4;
  const T* in = g + blockIdx.y * batch_stride;
  const int64_t packs = (columns + kSize - 1) / kSize, step = (int64_t)gridDim.x * kThreads;
  const int64_t first = (int64_t)blockIdx.x * kThreads + threadIdx.x, step_rows = step / packs, step_packs = step % packs;
  int64_t row = first / packs, pack = first % packs;
  float sum = 0.0f;
  auto advance = [&] {
    row += step_rows;
    pack += step_packs;
    if (pack >= packs) {
      pack -= packs;
      ++row;
    }
  };
  if (columns >= kSize) {
    // kOnce packs in flight; a row's last one ends with the row, and what it shares
    // with the one before counts there.
    while (row < rows) {
      Raw<T, kSize> v[kOnce];
      int counted[kOnce];  // from this element on
#pragma unroll
      for (int k = 0; k < kOnce; ++k) {
        const int64_t nominal = pack * kSize, at = nominal < columns - kSize ? nominal : columns - kSize;
        counted[k] = row < rows ? (int)(nominal - at) : kSize;
        v[k].load(in + (row < rows ? row * stride + at : 0));
        advance();
      }
#pragma unroll
      for (int k = 0; k < kOnce; ++k) {
        float x[kSize];
        v[k].get(x);
#pragma unroll
        for (int e = 0; e < kSize; ++e)
          if (e >= counted[k]) sum = fmaf(x[e], x[e], sum);
      }
    }
  } else {
    for (; row < rows; advance()) {
      float v[kSize];
      load_pack(in + row * stride, pack * kSize, columns, v);
#pragma unroll
      for (int e = 0; e < kSize; ++e) sum = fmaf(v[e], v[e], sum);
    }
  }
  sum = block_sum<kThreads>(sum, shared);
  if (threadIdx.x == 0) partial[blockIdx.y * kNormGroups + blockIdx.x] = sum;
}

// binary32 values are scaled to kScaleX X.  Those of 11 bits and fewer are scaled
// by a power of two alone, which leaves them what they are (their low parts are
// zero and never read); `rest`, 1 to 2, is what then takes them to kScaleX X.
struct Scaling {
  float scale, rest;
};

template <typename T>
__device__ __forceinline__ Scaling scale_for(float norm) {
  const float exact = kScaleX / norm;
  if constexpr (sizeof(T) == 4) return {exact, 1.0f};
  const float power = __uint_as_float(__float_as_uint(exact) & 0x7f800000u);
  return {power, power > 0.0f ? exact / power : exact};
}

// G as it lies and transposed, split and padded with zeros: 2,048 x 4,096 bfloat16
// 17 us, 84 MB; 1,500 x 1,001 binary32 7.6 us, and 11.2 with a load at a time.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_normalize(Split straight, Split turned, float* __restrict__ factor,
                                                        const T* __restrict__ g, const float* __restrict__ partial,
                                                        int64_t rows, int64_t columns, int64_t stride,
                                                        int64_t batch_stride, float eps) {
  __shared__ float shared[kThreads / kWave];
  __shared__ float tile[kPad][kPad + 1];
  const int64_t batch = blockIdx.z;
  const T* in = g + batch * batch_stride;
  const int64_t row0 = (int64_t)blockIdx.y * kPad, column0 = (int64_t)blockIdx.x * kPad;
  // All of a lane's values are on their way before the norm is known.
  constexpr int kRows = kThreads / kPad;
  const int x = threadIdx.x % kPad, y0 = threadIdx.x / kPad;
  T value[kPad / kRows];
#pragma unroll
  for (int k = 0; k < kPad / kRows; ++k) {
    const int64_t row = row0 + y0 + k * kRows;
    value[k] = in[row < rows && column0 + x < columns ? row * stride + column0 + x : 0];
  }
  const float norm = sqrtf(block_sum<kThreads>(partial[batch * kNormGroups + threadIdx.x], shared)) + eps;
  const Scaling scaling = scale_for<T>(norm);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) factor[batch] = scaling.rest;
#pragma unroll
  for (int k = 0; k < kPad / kRows; ++k) {
    const int y = y0 + k * kRows;
    tile[y][x] = row0 + y < rows && column0 + x < columns ? (float)value[k] * scaling.scale : 0.0f;
  }
  __syncthreads();
  // A lane takes four columns of four rows of each.
  for (int k = threadIdx.x; k < kPad * kPad / 4; k += kThreads) {
    const int y = k % kPad, from = k / kPad * 4;
    float4v a, b;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = tile[y][from + e];
      b[e] = tile[from + e][y];
    }
    store_four(element(straight, batch, (uint32_t)row0 + y, (uint32_t)column0 + from), a);
    store_four(element(turned, batch, (uint32_t)column0 + y, (uint32_t)row0 + from), b);
  }
}

// What a product becomes: symmetric results, of which only tiles on and above the
// diagonal are computed, alone or with the rest of a polynomial; a matrix and its
// transpose; the caller's result.
enum { kSymmetric, kPolynomial, kBoth, kFinal };
constexpr bool symmetric(int mode) { return mode == kSymmetric || mode == kPolynomial; }

struct Job {
  Split left, right;       // result = left right^T
  Split out, turned;       // symmetric: out; kBoth: out and its transpose
  Split added;             // kPolynomial: + added_factor added + diagonal I
  float added_factor, diagonal;
  float factor;            // of the sums,
  int powers;              // and this often given[batch]
};

struct Product {
  Job job[2];              // blockIdx.y: products of the same sizes
  const float* given;
  int64_t row_tiles, column_tiles, depth;  // of 32 rows; depth in blocks of 16
  void* result;            // kFinal: the caller's matrix, element (i, j) at i row_step + j column_step
  int64_t rows, columns, row_step, column_step, result_batch;
};

constexpr uint32_t kBand = 8;

// The tile of a workgroup: bands of kBand rows of tiles, column by column, and a
// share of that order to each chiplet (blockIdx.x modulo 8), so that what a
// chiplet works on at one time shares rows and columns in its cache.  Symmetric
// results have the tiles on and above the diagonal.
template <int kMode>
__device__ __forceinline__ bool find_tile(uint32_t row_tiles, uint32_t column_tiles, uint32_t* ti, uint32_t* tj) {
  uint32_t at = blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
  for (uint32_t first = 0; first < row_tiles; first += kBand) {
    const uint32_t count = kBand * (symmetric(kMode) ? column_tiles - first : column_tiles);
    if (at < count) {
      *ti = first + at % kBand;
      *tj = (symmetric(kMode) ? first : 0) + at / kBand;
      return *ti < row_tiles && (!symmetric(kMode) || *ti <= *tj);
    }
    at -= count;
  }
  return false;
}

// Where the four values of a lane belong in a tile's 32 x 32 (of tile (ti, tj)),
// and what they take.
template <int kMode, typename T>
struct Finish {
  const Product& p;
  _Float16 *turned, *straight;  // of the transposed tile, and of the tile
  const _Float16* old;
  T* final_to;
  float factor, added_factor, diagonal;
  bool mirrored, diagonal_tile;
  int64_t rows_left, columns_left;

  __device__ __forceinline__ Finish(const Product& product, const Job& job, int64_t batch, float total, uint32_t ti,
                                    uint32_t tj, bool off_diagonal)
      : p(product), factor(total), added_factor(job.added_factor), diagonal(job.diagonal),
        mirrored(kMode == kBoth || off_diagonal), diagonal_tile(ti == tj) {
    const int lane = threadIdx.x % kWave;
    if constexpr (kMode == kFinal) {
      const int64_t i = (int64_t)ti * 32 + lane / 32 * 4, j = (int64_t)tj * 32 + lane % 32;
      final_to = (T*)p.result + batch * p.result_batch + i * p.row_step + j * p.column_step;
      rows_left = p.rows - i;
      columns_left = p.columns - j;
    } else {
      turned = tile_of(kMode == kBoth ? job.turned : job.out, batch, tj, ti);
      straight = tile_of(job.out, batch, ti, tj);
      if constexpr (kMode == kPolynomial) old = tile_of(job.added, batch, tj, ti);  // symmetric
    }
  }
  // The added matrix' four, fetched before they are needed.
  __device__ __forceinline__ Parts fetch(int q) const {
    Parts parts = {};
    if constexpr (kMode == kPolynomial) {
      const _Float16* from = old + turned_place(threadIdx.x % kWave, q);
      parts.high = *(const half4*)from;
      parts.low = *(const half4*)(from + kBlock);
    }
    return parts;
  }
  __device__ __forceinline__ void operator()(int q, float4v v, const Parts& added) const {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= factor;
    if constexpr (kMode == kFinal) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (q * 8 + e < rows_left && columns_left > 0) final_to[(q * 8 + e) * p.row_step] = (T)v[e];
    } else {
      if constexpr (kMode == kPolynomial) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = fmaf(added_factor, (float)added.high[e] + (float)added.low[e], v[e]);
          v[e] += diagonal_tile && q * 8 + lane / 32 * 4 + e == lane % 32 ? diagonal : 0.0f;
        }
      }
      const Parts parts = parts_of(v);
      store_parts(turned + turned_place(lane, q), parts);
      if (mirrored) store_parts(straight + straight_place(lane, q), turn_quads(parts));
    }
  }
};

__device__ __forceinline__ float4v four_of(const float16v& v, int g) {
  return float4v{v[g * 4], v[g * 4 + 1], v[g * 4 + 2], v[g * 4 + 3]};
}

// sum += left right^T for a block each.
template <bool kLeftLow, bool kRightLow>
__device__ __forceinline__ void multiply_block(const half8* left, const half8* right, float16v& sum) {
  if constexpr (kRightLow) sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(left[0], right[1], sum, 0, 0, 0);
  if constexpr (kLeftLow) sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(left[1], right[0], sum, 0, 0, 0);
  sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(left[0], right[0], sum, 0, 0, 0);
}

__device__ __forceinline__ float total_factor(const Product& p, const Job& job, int64_t batch) {
  float factor = job.factor;
  for (int k = 0; k < job.powers; ++k) factor *= p.given[batch];
  return factor;
}

// Small products: a workgroup has a tile of 32 x 32, its kWaves waves a part of the
// depth each, joined in LDS.  Operands go from memory to registers, a ring of
// kAhead blocks, without a branch between a load and its use.  Bound by the launch
// and one walk along the depth: 4 to 6 us for sides of 512.
template <int kMode, typename T, int kWaves, bool kLeftLow, bool kRightLow>
__global__ __launch_bounds__(kWaves* kWave) void k_product_small(Product p) {
  constexpr int kAhead = 4;
  __shared__ float4v joined[kWaves > 1 ? kWaves * 4 * kWave : 1];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t batch = blockIdx.z;
  const Job& job = p.job[blockIdx.y];
  uint32_t ti, tj;
  if (!find_tile<kMode>((uint32_t)p.row_tiles, (uint32_t)p.column_tiles, &ti, &tj)) return;
  const half8* left = (const half8*)(job.left.data + batch * job.left.batch_stride + ti * job.left.blocks * 2 * kBlock) + lane;
  const half8* right = (const half8*)(job.right.data + batch * job.right.batch_stride + tj * job.right.blocks * 2 * kBlock) + lane;
  // What the end adds is fetched with the first operands.
  const Finish<kMode, T> finish(p, job, batch, total_factor(p, job, batch), ti, tj, ti != tj);
  constexpr int kMine = kWaves > 1 ? 1 : 4;  // quarters of the tile that a wave finishes
  Parts added[kMine];
#pragma unroll
  for (int q = 0; q < kMine; ++q) added[q] = finish.fetch(kWaves > 1 ? wave % 4 : q);
  struct Operands {
    half8 left[2], right[2];
  };
  auto fetch = [&](Operands& o, int64_t k) {
    o.left[0] = left[k * 2 * kWave];
    if constexpr (kLeftLow) o.left[1] = left[k * 2 * kWave + kWave];
    o.right[0] = right[k * 2 * kWave];
    if constexpr (kRightLow) o.right[1] = right[k * 2 * kWave + kWave];
  };
  // A sum for each kind of product: those of one sum wait for each other.
  float16v sums[3] = {};
  auto multiply = [&](const Operands& o) {
    sums[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(o.left[0], o.right[0], sums[0], 0, 0, 0);
    if constexpr (kLeftLow) sums[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(o.left[1], o.right[0], sums[1], 0, 0, 0);
    if constexpr (kRightLow) sums[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(o.left[0], o.right[1], sums[2], 0, 0, 0);
  };
  const int64_t share = (p.depth + kWaves - 1) / kWaves, begin = wave * share;
  const int64_t steps = (begin + share < p.depth ? begin + share : p.depth) - begin;
  if (steps > 0) {
    Operands ring[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) fetch(ring[q], begin + (q < steps ? q : steps - 1));
    int64_t k = 0;
    for (; k + kAhead <= steps; k += kAhead)
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        multiply(ring[q]);
        const int64_t ahead = k + q + kAhead;
        fetch(ring[q], begin + (ahead < steps ? ahead : steps - 1));
      }
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (k + q < steps) multiply(ring[q]);
  }
  float16v sum = sums[0];
  if constexpr (kLeftLow || kRightLow) sum += sums[1] + sums[2];
  if constexpr (kWaves > 1) {
    // The first four waves join and finish a quarter each.
#pragma unroll
    for (int q = 0; q < 4; ++q) joined[(wave * 4 + q) * kWave + lane] = four_of(sum, q);
    __syncthreads();
    if (wave >= 4) return;
    float4v v = joined[wave * kWave + lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += joined[(w * 4 + wave) * kWave + lane];
    finish(wave, v, added[0]);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) finish(q, four_of(sum, q), added[kWaves > 1 ? 0 : q]);
  }
}

using GlobalBytes = const __attribute__((address_space(1))) void*;
using SharedBytes = __attribute__((address_space(3))) void*;

// Large products: a tile of 64 kHalf x 64 kHalf, kHalf x kHalf blocks of 32 to each
// of four waves.  What a compute unit gets from its chiplet's cache bounds
// products of this kind (34 bytes a clock measured, where registers alone carry
// them), so the waves share their operands in LDS.  Stages of kDepth blocks of 16
// are loaded straight into a ring of kRing in LDS, a block as it lies in memory,
// a lane's 16 bytes at 16 lane; a wave reads a stage into registers while it
// multiplies the one before.  2,048^3 of three instructions: symmetric 44 us (136
// tiles, so 120 of 256 compute units stand idle; a half of its loop's time is the
// matrix instructions', the rest waits for LDS's loads), 1,024 with tiles of 64 14;
// 2,048 x 2,048 x 4,096 of three, whose tiles are two to a compute unit in turns,
// 96 us, 1,070 TFLOP/s.  With four waves more that do nothing but load: 4 % slower.
template <int kMode, typename T, int kHalf, bool kLeftLow, bool kRightLow>
__global__ __launch_bounds__(4 * kWave, 1) void k_product(Product p) {
  constexpr int kRing = 4, kDepth = 4 / kHalf;
  constexpr int kSide = 2 * kHalf;  // blocks of the tile on either side
  constexpr int kLeft = kSide * (1 + kLeftLow), kRight = kSide * (1 + kRightLow);  // blocks of one depth
  constexpr int kLoads = (kLeft + kRight) * kDepth / 4;  // of a wave and stage
  constexpr int kStage = (kLeft + kRight) * kDepth * kBlock;
  __shared__ __attribute__((aligned(1024))) _Float16 stages[kRing][kStage];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t batch = blockIdx.z;
  const Job& job = p.job[blockIdx.y];
  uint32_t ti, tj;
  if (!find_tile<kMode>((uint32_t)(p.row_tiles / kSide), (uint32_t)(p.column_tiles / kSide), &ti, &tj)) return;
  // What the end adds is fetched first.
  constexpr int kSums = kHalf * kHalf;
  const float factor = total_factor(p, job, batch);
  auto finish_of = [&](int s) {
    return Finish<kMode, T>(p, job, batch, factor, ti * kSide + wave / 2 * kHalf + s / kHalf, tj * kSide + wave % 2 * kHalf + s % kHalf, ti != tj);
  };
  Parts added[kSums][4];
#pragma unroll
  for (int s = 0; s < kSums; ++s)
#pragma unroll
    for (int q = 0; q < 4; ++q) added[s][q] = finish_of(s).fetch(q);
  // The blocks this wave loads of every stage.
  const _Float16* from[kLoads];
#pragma unroll
  for (int q = 0; q < kLoads; ++q) {
    const int b = q * 4 + wave, d = b / (kLeft + kRight), in = b % (kLeft + kRight);
    const bool is_left = in < kLeft;
    const int c = is_left ? in : in - kLeft;
    const Split& m = is_left ? job.left : job.right;
    from[q] = m.data + batch * m.batch_stride + ((int64_t)((is_left ? ti : tj) * kSide + c % kSide) * m.blocks + d) * (2 * kBlock) +
              c / kSide * kBlock + lane * 8;
  }
  const int64_t steps = p.depth / kDepth;
  // Steps beyond the last are loaded (again) and not multiplied: the count of
  // loads in flight stays what the waits below take it for.
  auto load = [&](int64_t step, int q) {
    const int64_t at = (step < steps ? step : steps - 1) * (kDepth * 2 * kBlock);
    __builtin_amdgcn_global_load_lds((GlobalBytes)(from[q] + at),
                                     (SharedBytes)(stages[step % kRing] + (q * 4 + wave) * kBlock), 16, 0, 0);
  };
  // Until this wave's loads of the oldest of three stages in flight are there and
  // its reads of LDS done; then until the other waves' are.
  auto arrived = [&] {
    constexpr int kFlight = 2 * kLoads;
    static_assert(kFlight < 64, "vmcnt");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x70 | (kFlight & 15) | (kFlight >> 4) << 14);  // vmcnt(kFlight) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // A stage's operands in registers: [side][depth][block][high, low].
  struct Operands {
    half8 v[2][kDepth][kHalf][2];
  };
  const int wi = wave / 2 * kHalf, wj = wave % 2 * kHalf;
  constexpr int kEach = kDepth * kHalf, kReads = kEach * (2 + kLeftLow + kRightLow);
  auto read = [&](Operands& o, int64_t step, int r) {
    const int high = r < 2 * kEach, side = high ? r / kEach : kLeftLow && r < 3 * kEach ? 0 : 1;
    const int d = r % kEach / kHalf, i = r % kHalf;
    const half8* blocks = (const half8*)stages[step % kRing] + lane;
    o.v[side][d][i][1 - high] = blocks[(d * (kLeft + kRight) + (side ? kLeft + wj : wi) + i + (high ? 0 : kSide)) * kWave];
  };
  // The instructions of a stage, those on one sum far apart.
  constexpr int kProducts = 1 + kLeftLow + kRightLow, kCalls = kProducts * kDepth * kSums;
  constexpr int kChains = kSums < 4 ? 2 : 1;  // sums of a block, where the blocks are few
  float16v sum[kSums][kChains] = {};
  auto multiply = [&](const Operands& o, int t) {
    const int s = t % kSums, d = t / kSums % kDepth, product = t / (kSums * kDepth);
    const int low_left = kLeftLow && product == 1, low_right = kRightLow && product == 1 + kLeftLow;
    sum[s][t / kSums % kChains] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
        o.v[0][d][s / kHalf][low_left], o.v[1][d][s % kHalf][low_right], sum[s][t / kSums % kChains], 0, 0, 0);
  };
  for (int q = 0; q < kRing; ++q)
#pragma unroll
    for (int l = 0; l < kLoads; ++l) load(q, l);
  Operands ring[2];
  __builtin_amdgcn_s_waitcnt(0x70 | (3 * kLoads & 15) | (3 * kLoads >> 4) << 14);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int r = 0; r < kReads; ++r) read(ring[0], 0, r);
  // A step: its operands are in registers; the next one's are read from LDS and the
  // stage it was read from itself is loaded anew (every wave has reached the
  // barrier with its reads of that stage done) between the multiplications, as
  // many of these after each load as keep a wave from waiting to issue it.
  constexpr int kPer = kCalls / kLoads;
  for (int64_t step = 0; step < steps; step += 2) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t here = step + q;
      if (q == 1 && here >= steps) break;
      arrived();
#pragma unroll
      for (int t = 0; t < kCalls; ++t) {
        if (t % kPer == 0) {
          __builtin_amdgcn_sched_barrier(0);
          if (t / kPer < kLoads) load(here + kRing, t / kPer);
#pragma unroll
          for (int more = 0; more < (kReads + kLoads - 1) / kLoads; ++more)
            if (t / kPer * ((kReads + kLoads - 1) / kLoads) + more < kReads)
              read(ring[1 - q], here + 1, t / kPer * ((kReads + kLoads - 1) / kLoads) + more);
          __builtin_amdgcn_sched_barrier(0);
        }
        multiply(ring[q], t);
      }
    }
  }
  // Nothing may land in LDS after the workgroup has ended.
  __builtin_amdgcn_s_waitcnt(0x70);  // vmcnt(0) lgkmcnt(0)
#pragma unroll
  for (int s = 0; s < kSums; ++s) {
    if constexpr (kChains > 1) sum[s][0] += sum[s][1];
    const Finish<kMode, T> finish = finish_of(s);
#pragma unroll
    for (int q = 0; q < 4; ++q) finish(q, four_of(sum[s][0], q), added[s][q]);
  }
}

// One workgroup for a whole matrix of at most 64 rows (after transposition): the
// m x m matrices stay in LDS, X and its transpose in the workspace, where they
// are in this compute unit's cache, and nothing waits for a launch: 64 x 256 50 us,
// by launches 77.
constexpr int kOneSide = 64, kOneThreads = 512, kOneWaves = kOneThreads / kWave;
constexpr int kSquare = kOneSide * kOneSide * 2;      // halves of a matrix in LDS
constexpr int kJoined = kOneWaves / 2 * 3 * 4 * kWave;  // float4s of the partial sums of A

template <typename T>
__global__ __launch_bounds__(kOneThreads) void k_one(T* __restrict__ out, const T* __restrict__ g, Split x, Split xt,
                                                     Split xt_next, int64_t rows, int64_t columns, int64_t stride,
                                                     int64_t batch_stride, int steps, int most, float a, float b,
                                                     float c, float eps) {
  constexpr bool kExact = sizeof(T) == 2;
  constexpr int kSize = Pack<T>::kSize;
  // A apart: its partial sums lie where the others will.
  constexpr int kA = 4 * kSquare;
  static_assert(kJoined * 8 <= kA, "the partial sums fit the others' place");
  __shared__ __attribute__((aligned(1024))) _Float16 lds[kA + kSquare];
  __shared__ float shared[kOneWaves];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t batch = blockIdx.x;
  const bool tall = rows > columns;
  const int64_t m = tall ? columns : rows, n = tall ? rows : columns, np = x.blocks * 16;
  const T* in = g + batch * batch_stride;

  float squares = 0.0f, v[kSize];
  const int64_t packs = (columns + kSize - 1) / kSize;
  for (int64_t i = threadIdx.x; i < rows * packs; i += kOneThreads) {
    const int64_t row = i / packs;
    load_pack(in + row * stride, (i - row * packs) * kSize, columns, v);
#pragma unroll
    for (int e = 0; e < kSize; ++e) squares = fmaf(v[e], v[e], squares);
  }
  const Scaling scaling = scale_for<T>(sqrtf(block_sum<kOneThreads>(squares, shared)) + eps);

  // X and X^T, a 4 x 4 at a time; lanes follow each other along G's rows.
  const uint32_t quads = (uint32_t)np / 4;
  for (uint32_t k = threadIdx.x; k < kOneSide / 4 * quads; k += kOneThreads) {
    const uint32_t i = (tall ? k % (kOneSide / 4) : k / quads) * 4, j = (tall ? k / (kOneSide / 4) : k % quads) * 4;
    const int64_t down = tall ? 1 : stride, across = tall ? stride : 1;
    const T* from = in + i * down + j * across;
    float4v straight[4], turned[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float value = i + r < m && j + e < n ? (float)from[r * down + e * across] * scaling.scale : 0.0f;
        straight[r][e] = value;
        turned[e][r] = value;
      }
    _Float16 *first = element(x, batch, i, j), *first_turned = element(xt, batch, j, i);
#pragma unroll
    for (int r = 0; r < 4; ++r) {  // rows of a block follow each other at 8 halves
      store_four(first + r * 8, straight[r]);
      store_four(first_turned + r * 8, turned[r]);
    }
  }
  __syncthreads();

  int Z = 0, U = kSquare, P = 2 * kSquare, Q = 3 * kSquare;
  auto block_at = [&](int matrix, int row_tile, int k) {
    return (const half8*)(lds + matrix + (row_tile * (kOneSide / 16) + k) * 2 * kBlock) + lane;
  };
  auto square_tile = [&](int matrix, int row_tile, int column_tile) {
    return lds + matrix + (row_tile * (kOneSide / 16) + 2 * column_tile) * (2 * kBlock);
  };
  // A tile of left right^T (0: upper left, 1: upper right, 2: lower right) by a wave;
  // one sum for each kind of product, so that four depths follow each other, not twelve.
  auto square = [&](int tile, int left, int right, int to, float factor, bool added) {
    const int ti = tile / 2, tj = (tile + 1) / 2;
    float16v sum[3] = {};
#pragma unroll
    for (int k = 0; k < kOneSide / 16; ++k) {
      const half8 *l = block_at(left, ti, k), *r = block_at(right, tj, k);
      sum[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[0], r[0], sum[0], 0, 0, 0);
      sum[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[kWave], r[0], sum[1], 0, 0, 0);
      sum[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[0], r[kWave], sum[2], 0, 0, 0);
    }
    sum[0] += sum[1] + sum[2];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float4v w = four_of(sum[0], q);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] *= factor;
      if (added) {
        const float4v old = load_four(square_tile(kA, tj, ti) + turned_place(lane, q));
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = fmaf(b * kScaleZ / kScaleX, old[e], w[e]);
        if (ti == tj)
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] += q * 8 + lane / 32 * 4 + e == lane % 32 ? a * kScaleZ : 0.0f;
      }
      const Parts parts = parts_of(w);
      store_parts(square_tile(to, tj, ti) + turned_place(lane, q), parts);
      if (ti != tj) store_parts(square_tile(to, ti, tj) + straight_place(lane, q), turn_quads(parts));
    }
  };

  const int segments = (steps + most - 1) / most;
  for (int s = 0; s < segments; ++s) {
    const int length = steps / segments + (s < steps % segments ? 1 : 0);
    const bool exact = kExact && s == 0, last = s + 1 == segments;
    // A = X X^T: every wave some depths of all three tiles.
    {
      float16v sum[3] = {};
      const half8* from = (const half8*)(x.data + batch * x.batch_stride) + lane;
#pragma unroll 2
      for (int64_t k = wave; k < x.blocks; k += kOneWaves) {
        half8 top[2], bottom[2];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          top[part] = from[(k * 2 + part) * kWave];
          bottom[part] = from[((x.blocks + k) * 2 + part) * kWave];
        }
        multiply_block<true, true>(top, top, sum[0]);
        multiply_block<true, true>(top, bottom, sum[1]);
        multiply_block<true, true>(bottom, bottom, sum[2]);
      }
      float4v* joined = (float4v*)lds;
      const int slot = wave % (kOneWaves / 2);
      for (int half = 1; half >= 0; --half) {
        if (wave / (kOneWaves / 2) == half)
#pragma unroll
          for (int t = 0; t < 3; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              float4v& at = joined[((t * 4 + q) * (kOneWaves / 2) + slot) * kWave + lane];
              at = half ? four_of(sum[t], q) : at + four_of(sum[t], q);
            }
        __syncthreads();
      }
      for (int part = wave; part < 12; part += kOneWaves) {
        const int tile = part / 4, q = part % 4, ti = tile / 2, tj = (tile + 1) / 2;
        float4v w = joined[part * (kOneWaves / 2) * kWave + lane];
#pragma unroll
        for (int k = 1; k < kOneWaves / 2; ++k) w += joined[(part * (kOneWaves / 2) + k) * kWave + lane];
        const float factor = exact ? scaling.rest * scaling.rest / kScaleX : 1.0f / kScaleX;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] *= factor;
        const Parts parts = parts_of(w);
        store_parts(square_tile(kA, tj, ti) + turned_place(lane, q), parts);
        if (ti != tj) store_parts(square_tile(kA, ti, tj) + straight_place(lane, q), turn_quads(parts));
      }
      __syncthreads();
    }
    for (int k = 0; k < length; ++k) {
      // Z; then U <- Z A and (but Z itself is P at first) Q <- Z P side by side; then
      // A <- U Z.  One copy of the code: what is fetched once only costs more than
      // it computes.
      const bool more = k + 1 < length;
#pragma unroll 1
      for (int phase = 0; phase < 3; ++phase) {
        const bool second = wave >= 3;
        const bool runs = phase == 0 ? !second : phase == 1 ? (second ? k > 0 : more) : !second && more;
        if (wave < 6 && runs)
          square(wave % 3, phase == 0 ? kA : phase == 1 ? Z : U, phase == 2 ? Z : second ? P : kA,
                 phase == 0 ? Z : phase == 1 ? (second ? Q : U) : kA,
                 phase == 0 ? c * kScaleZ / (kScaleX * kScaleX) : 1.0f / kScaleZ, phase == 0);
        __syncthreads();
      }
      const int next = k == 0 ? Z : Q;
      (k == 0 ? Z : Q) = P;
      P = next;
    }
    // X = P X, a tile of 32 x 32 a wave.
    const float factor = (exact ? scaling.rest : 1.0f) / (last ? kScaleZ * kScaleX : kScaleZ);
    for (uint32_t t = wave; t < 2 * (uint32_t)(np / 32); t += kOneWaves) {
      const uint32_t ti = t % 2, tj = t / 2;
      const half8* from = (const half8*)(xt.data + batch * xt.batch_stride + tj * xt.blocks * 2 * kBlock) + lane;
      float16v sum[3] = {};
      half8 right[kOneSide / 16][2];
#pragma unroll
      for (int k = 0; k < kOneSide / 16; ++k) {
        right[k][0] = from[k * 2 * kWave];
        right[k][1] = from[k * 2 * kWave + kWave];
      }
#pragma unroll
      for (int k = 0; k < kOneSide / 16; ++k) {
        const half8* l = block_at(P, ti, k);
        sum[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[0], right[k][0], sum[0], 0, 0, 0);
        sum[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[kWave], right[k][0], sum[1], 0, 0, 0);
        sum[2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l[0], right[k][1], sum[2], 0, 0, 0);
      }
      sum[0] += sum[1] + sum[2];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float4v w = four_of(sum[0], q);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] *= factor;
        if (last) {
          const int64_t i = ti * 32 + q * 8 + lane / 32 * 4, j = tj * 32 + lane % 32;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < m && j < n)
              out[batch * rows * columns + (tall ? j * columns + i + e : (i + e) * columns + j)] = (T)w[e];
        } else {
          const Parts parts = parts_of(w);
          store_parts(tile_of(xt_next, batch, tj, ti) + turned_place(lane, q), parts);
          store_parts(tile_of(x, batch, ti, tj) + straight_place(lane, q), turn_quads(parts));
        }
      }
    }
    __syncthreads();
    const Split now = xt;
    xt = xt_next;
    xt_next = now;
  }
}

// ---- host -------------------------------------------------------------------

// Whole tiles of 64, of 128 where those are taken.
int64_t padded(int64_t v) {
  const int64_t to = v > 1024 ? 2 * kPad : kPad;
  return (v + to - 1) / to * to;
}

// The largest |f(t)| of t in [0, end], where f' has the roots of u + v t + w t^2.
template <typename F>
double largest(F&& f, double end, double u, double v, double w) {
  double most = std::fmax(std::fabs(f(0.0)), std::fabs(f(end)));
  auto at = [&](double t) {
    if (t > 0.0 && t < end) most = std::fmax(most, std::fabs(f(t)));
  };
  const double d = v * v - 4.0 * u * w;
  if (d < 0.0) return most;
  const double q = -0.5 * (v + std::copysign(std::sqrt(d), v));
  if (w != 0.0) at(q / w);
  if (q != 0.0) at(u / q);
  return most;
}

// Whether all matrices stay within what their scales let binary16 hold.  Each is a
// polynomial of X's singular values, which begin within [0, 1]; no entry is larger
// than the largest singular value.  With `most` steps a segment.
bool in_range(int steps, int most, double a, double b, double c) {
  const double most_x = kMostHalf / kScaleX, most_z = kMostHalf / kScaleZ;
  auto z = [&](double t) { return a + b * t + c * t * t; };  // t: eigenvalues of A
  double end = 1.0, before[2] = {1.0, 1.0};                  // of A; of the steps before, Z's largest
  for (int k = 0; k < steps; ++k) {
    if (end > most_x) return false;  // A, and X with it
    const double now = largest(z, end, b, 2.0 * c, 0.0);
    if (now > most_z || (most > 1 && now * before[0] * before[1] > most_z)) return false;  // Z; P
    if (k + 1 == steps) break;  // (the last step's result is the caller's)
    if (most > 1 && largest([&](double t) { return t * z(t); }, end, a, 2.0 * b, 3.0 * c) > most_x) return false;  // U
    const double s = largest([&](double t) { return std::sqrt(t) * z(t); }, end, a, 3.0 * b, 5.0 * c);
    end = s * s;
    before[1] = before[0];
    before[0] = now;
  }
  return true;
}

// The longer side up to which one workgroup takes a matrix of kOneSide rows.  Measured
// with binary32, us: 64 x 256 51 and 77, 64 x 512 82 and 78.
constexpr int64_t kOneLength = 448;

// Where the matrices lie in the workspace.
struct Plan {
  int64_t m, n, mp, np;
  size_t partial, factor, x, xt, xt_next, square[5], bytes;
};

Plan plan(int64_t batch, int64_t rows, int64_t columns) {
  Plan p = {};
  p.m = rows < columns ? rows : columns;
  p.n = rows < columns ? columns : rows;
  p.mp = padded(p.m);
  p.np = padded(p.n);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t from = at;
    at += (bytes + 255) / 256 * 256;
    return from;
  };
  p.partial = take((size_t)batch * kNormGroups * sizeof(float));
  p.factor = take((size_t)batch * sizeof(float));
  const size_t wide = (size_t)batch * p.mp * p.np * 2 * sizeof(_Float16);
  p.x = take(wide);
  p.xt = take(wide);
  p.xt_next = take(wide);
  for (auto& s : p.square) s = take((size_t)batch * p.mp * p.mp * 2 * sizeof(_Float16));
  p.bytes = at;
  return p;
}

// Workgroups for tiles of `side` blocks: whole eights, so that every chiplet's
// share of find_tile's order has the same length.
template <int kMode>
dim3 product_grid(const Product& p, int side, int jobs, int64_t batch) {
  const int64_t rows = p.row_tiles / side, columns = p.column_tiles / side;
  int64_t tiles = 0;
  for (int64_t first = 0; first < rows; first += kBand) tiles += kBand * (symmetric(kMode) ? columns - first : columns);
  return dim3((uint32_t)((tiles + 7) / 8 * 8), (uint32_t)jobs, (uint32_t)batch);
}

// Tiles of 128 where they are enough for half the compute units, of 64 where those
// are enough for a quarter, else of 32 with the depth cut into parts.  us by this rule
// and otherwise: 2,048 x 4,096 bfloat16 881, with tiles of 64 alone 955; 1,024 x 1,024
// binary32 174, with 128 from 64 tiles on 222; 1,900 x 2,100 824, with 128 from 100 on
// 798; 1,500 x 1,001 224, without tiles of 64 386; 512 x 512 97, with 64 from 32 tiles on
// 124, from 100 on 87; 8 of 512 x 512 258 and 253 without tiles of 64.  Parts of the
// depth: 512 x 512 97, in one up to a depth of 1,024 115, in 16 always 103, in 4 beyond
// 256 98; 128 x 1,000 78, in 4 beyond 256 71.
template <int kMode, typename T, bool kLeftLow, bool kRightLow>
void product(const Product& p, int jobs, int64_t batch, hipStream_t stream) {
  auto tiles = [&](int side) {
    const int64_t rows = p.row_tiles / side, columns = p.column_tiles / side;
    return (symmetric(kMode) ? rows * (rows + 1) / 2 : rows * columns) * jobs * batch;
  };
  auto small = [&](auto waves) {
    constexpr int kWaves = decltype(waves)::value;
    hipLaunchKernelGGL((k_product_small<kMode, T, kWaves, kLeftLow, kRightLow>), product_grid<kMode>(p, 1, jobs, batch),
                       dim3(kWaves * kWave), 0, stream, p);
  };
  if (p.row_tiles % 4 == 0 && p.column_tiles % 4 == 0 && tiles(4) >= 128)
    hipLaunchKernelGGL((k_product<kMode, T, 2, kLeftLow, kRightLow>), product_grid<kMode>(p, 4, jobs, batch),
                       dim3(4 * kWave), 0, stream, p);
  else if (tiles(2) >= 64 && p.depth >= 16)
    hipLaunchKernelGGL((k_product<kMode, T, 1, kLeftLow, kRightLow>), product_grid<kMode>(p, 2, jobs, batch),
                       dim3(4 * kWave), 0, stream, p);
  else if (p.depth < 16) small(std::integral_constant<int, 1>());
  else if (p.depth < 64) small(std::integral_constant<int, 4>());
  else small(std::integral_constant<int, 16>());
}

template <typename T>
int orthogonalize(T* out, const T* g, int64_t batch, int64_t rows, int64_t columns, int64_t stride,
                  int64_t batch_stride, int steps, float a, float b, float c, float eps, uint8_t* ws,
                  hipStream_t stream) {
  constexpr bool kExact = sizeof(T) == 2;  // X0 has no low parts
  const Plan pl = plan(batch, rows, columns);
  const bool tall = rows > columns;
  float *partial = (float*)(ws + pl.partial), *factor = (float*)(ws + pl.factor);
  auto matrix = [&](size_t at, int64_t r, int64_t s) { return Split{(_Float16*)(ws + at), s / 16, r * s * 2}; };
  const Split x = matrix(pl.x, pl.mp, pl.np);
  Split xt = matrix(pl.xt, pl.np, pl.mp), xt_next = matrix(pl.xt_next, pl.np, pl.mp);
  Split A = matrix(pl.square[0], pl.mp, pl.mp), Z = matrix(pl.square[1], pl.mp, pl.mp),
        U = matrix(pl.square[2], pl.mp, pl.mp), P = matrix(pl.square[3], pl.mp, pl.mp),
        Q = matrix(pl.square[4], pl.mp, pl.mp);
  constexpr int kMost = kExact ? kSegment16 : kSegment32;
  if (pl.m <= kOneSide && pl.n <= kOneLength) {
    hipLaunchKernelGGL((k_one<T>), dim3((uint32_t)batch), dim3(kOneThreads), 0, stream, out, g, x, xt, xt_next, rows,
                       columns, stride, batch_stride, steps, kMost, a, b, c, eps);
    MGB_LAUNCH_CHECK("orthogonalize: one workgroup");
    return 0;
  }
  hipLaunchKernelGGL((k_square_sums<T>), dim3(kNormGroups, (uint32_t)batch), dim3(kThreads), 0, stream, partial, g, rows,
                     columns, stride, batch_stride);
  hipLaunchKernelGGL((k_normalize<T>),
                     dim3((uint32_t)(padded(columns) / kPad), (uint32_t)(padded(rows) / kPad), (uint32_t)batch),
                     dim3(kThreads), 0, stream, tall ? xt : x, tall ? x : xt, factor, g, partial, rows, columns, stride,
                     batch_stride, eps);
  MGB_LAUNCH_CHECK("orthogonalize: scaling");
  Product square = {};  // m x m results
  square.given = factor;
  square.row_tiles = square.column_tiles = pl.mp / 32;
  square.depth = pl.mp / 16;
  auto job = [&](Split left, Split right, Split to, float scale) {
    Job j = {};
    j.left = left;
    j.right = right;
    j.out = to;
    j.factor = scale;
    return j;
  };
  // Segments of one step (the products as they stand in the formula) take three
  // launches a step, of three steps 3.3, and multiplications with n in every step.
  // Measured with bfloat16, us: 1,500 x 2,048 461 and 464, 700 x 1,400 201 and 184;
  // 128 x 1,000 88 and 90, 128 x 2,048 101 and 93.
  const bool plain = 5 * pl.n <= 7 * pl.m || (pl.m <= 384 && pl.n <= 1024);
  const int most = plain ? 1 : kMost, segments = (steps + most - 1) / most;
  for (int s = 0; s < segments; ++s) {
    const int length = steps / segments + (s < steps % segments ? 1 : 0);
    Product gram = square;
    gram.job[0] = job(x, x, A, 1.0f / kScaleX);
    gram.depth = pl.np / 16;
    if (kExact && s == 0) {
      gram.job[0].powers = 2;
      product<kSymmetric, float, false, false>(gram, 1, batch, stream);
    } else {
      product<kSymmetric, float, true, true>(gram, 1, batch, stream);
    }
    for (int k = 0; k < length; ++k) {
      square.job[0] = job(A, A, Z, c * kScaleZ / (kScaleX * kScaleX));
      square.job[0].added = A;
      square.job[0].added_factor = b * kScaleZ / kScaleX;
      square.job[0].diagonal = a * kScaleZ;
      product<kPolynomial, float, true, true>(square, 1, batch, stream);
      // P <- Z P (Z itself at first) and U <- Z A side by side, then A <- U Z.
      int jobs = 0;
      if (k > 0) square.job[jobs++] = job(Z, P, Q, 1.0f / kScaleZ);
      if (k + 1 < length) square.job[jobs++] = job(Z, A, U, 1.0f / kScaleZ);
      if (jobs) product<kSymmetric, float, true, true>(square, jobs, batch, stream);
      if (k + 1 < length) {
        square.job[0] = job(U, Z, A, 1.0f / kScaleZ);
        product<kSymmetric, float, true, true>(square, 1, batch, stream);
      }
      if (k == 0) std::swap(P, Z);
      else std::swap(P, Q);
    }
    Product wide = {};
    wide.given = factor;
    wide.row_tiles = pl.mp / 32;
    wide.column_tiles = pl.np / 32;
    wide.depth = pl.mp / 16;
    const bool first = kExact && s == 0, last = s + 1 == segments;
    wide.job[0] = job(P, xt, x, last ? 1.0f / (kScaleZ * kScaleX) : 1.0f / kScaleZ);
    wide.job[0].powers = first ? 1 : 0;
    // X^T is read whole while the new one is written: two buffers in turn.
    wide.job[0].turned = xt_next;
    wide.result = out;
    wide.rows = pl.m;
    wide.columns = pl.n;
    wide.row_step = tall ? 1 : columns;
    wide.column_step = tall ? columns : 1;
    wide.result_batch = rows * columns;
    if (last && first) product<kFinal, T, true, false>(wide, 1, batch, stream);
    else if (last) product<kFinal, T, true, true>(wide, 1, batch, stream);
    else if (first) product<kBoth, float, true, false>(wide, 1, batch, stream);
    else product<kBoth, float, true, true>(wide, 1, batch, stream);
    std::swap(xt, xt_next);
  }
  MGB_LAUNCH_CHECK("orthogonalize: products");
  return 0;
}

}  // namespace
}  // namespace mgb

using namespace mgb;

extern "C" {

size_t mgb_orthogonalize_workspace_bytes(int64_t batch, int64_t rows, int64_t columns) {
  if (batch < 1 || rows < 1 || columns < 1 || rows > kMostSide || columns > kMostSide) return 0;
  return plan(batch, rows, columns).bytes;
}

int mgb_orthogonalize(void* out, const void* update, int64_t batch, int64_t rows, int64_t columns, int64_t stride,
                      int64_t batch_stride, int steps, const float* coefficients, float eps, int dtype, void* workspace,
                      size_t workspace_bytes, void* stream) {
  MGB_REQUIRE(batch >= 0 && batch < 65536, "orthogonalize: at most 65,535 matrices");
  MGB_REQUIRE(rows >= 0 && columns >= 0 && rows <= kMostSide && columns <= kMostSide,
              "orthogonalize: a matrix' sides must be at most 2^20");
  MGB_REQUIRE(steps >= 1 && steps <= 100, "orthogonalize: steps must be 1 to 100");
  MGB_REQUIRE(coefficients, "orthogonalize: null pointer");
  for (int k = 0; k < 3; ++k)
    MGB_REQUIRE(coefficients[k] >= -kMostCoefficient && coefficients[k] <= kMostCoefficient,
                "orthogonalize: coefficients must lie within -8 and 8");
  MGB_REQUIRE(eps >= 0.0f, "orthogonalize: eps must not be negative");
  if (batch == 0 || rows == 0 || columns == 0) return 0;
  MGB_REQUIRE(out && update && workspace, "orthogonalize: null pointer");
  MGB_REQUIRE(workspace_bytes >= mgb_orthogonalize_workspace_bytes(batch, rows, columns),
              "orthogonalize: workspace too small");
  auto run = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    MGB_REQUIRE(in_range(steps, sizeof(T) == 4 ? kSegment32 : kSegment16, coefficients[0], coefficients[1],
                         coefficients[2]),
                "orthogonalize: with these coefficients and steps a singular value of at most 1 may grow beyond what "
                "the products hold (about 4)");
    return orthogonalize<T>((T*)out, (const T*)update, batch, rows, columns, stride, batch_stride, steps,
                            coefficients[0], coefficients[1], coefficients[2], eps, (uint8_t*)workspace,
                            (hipStream_t)stream);
  };
  switch (dtype) {
    case MGB_F32: return run((float*)nullptr);
    case MGB_F16: return run((_Float16*)nullptr);
    case MGB_BF16: return run((__bf16*)nullptr);
  }
  set_error("orthogonalize: types must be float32, float16 or bfloat16");
  return -1;
}

}  // extern "C"
