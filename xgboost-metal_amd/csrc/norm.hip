// Layer norm over the last axis and its gradient.
//
//   mean = sum x / D,  rstd = (sum (x - mean)^2 / D + eps)^-1/2
//   y = (x - mean) rstd w + b
// and, with h = (x - mean) rstd and g = dy w,
//   dx = rstd (g - sum g / D - h sum(g h) / D),  dw = sum_rows dy h,  db = sum_rows dy.
//
// Both passes are bound by memory: a row is read once into registers by the
// lanes that hold it (a part of a wave, a wave or a workgroup, by its width),
// the sums go over those lanes, and the row is written from the registers.
// All sums are binary32.  A mean rounded to it is off by up to an ulp or more, which
// in a row far from zero is more than its spread, so the centred values are summed
// once more: what is left of the mean is taken out of them, of the variance (a sum of
// centred squares, not a difference of sums) and of the stored mean.  The gradient
// centres by the stored mean, half an ulp of it off at most: h there is off by that
// times rstd, 2^-13 where a row's spread is 2^12 ulps of its mean.
//
// Measured (us, one MI355X, whose copies reach 5.1 TB/s), with the bytes that
// have to move: 65,536 x 1,024 bfloat16 forward 54 (5.0 TB/s), gradient 74 and the
// joining of its column sums 5 (5.1 TB/s); 5,003 x 1,000 binary32 gradient 13 and
// 4 (3.6 TB/s: the second launch, and eight waves a CU with 2.4 rows each); 16 x 32
// 1.9, a launch.
#include <type_traits>

#include "encoder_common.hpp"

namespace mgb {
namespace {

constexpr int kNormThreads = 256;
// Of the gradient's workgroups: several rows where a row is at most a wave's, else
// one (its sums take the whole workgroup's barriers).
constexpr int gradient_threads(int lanes) { return lanes > kWave ? lanes : 512; }
constexpr int kReduceColumns = 32, kReduceSlices = 32;

// Elements a lane holds at most, in a row of a wave and in one of a workgroup; beyond
// 256 lanes 1024 take a row, and rows wider still are read again for each sum.
// Measured with 33 million values in all (us, forward and gradient): binary32 rows of
// 1,024 by a wave 44 and 49, by 256 lanes 46 and 65; of 2,048 by 256 lanes 42 and 53,
// by a wave 48 and 126; of 4,096 by 256 lanes 44 and 52, by 1024 50 and 54; bfloat16
// rows of 8,192 by 256 lanes 26 and 50, by 1024 31 and 42; binary32 rows of 16,384 from
// registers 50 and 139, read again 79 and 205; of 32,768 62 and 82 (forward).
constexpr int kWaveElements = 16, kBlockElements = 32;

// Sum over the kLanes that share a row.
template <int kLanes>
__device__ __forceinline__ float row_sum(float v, float* shared) {
  if constexpr (kLanes <= kWave) {
    return group_sum<kLanes>(v);
  } else {
    return block_sum<kLanes>(v, shared);
  }
}

template <int kLanes>
__device__ __forceinline__ void row_sums(float& a, float& b, float* shared) {
  if constexpr (kLanes <= kWave) {
    a = group_sum<kLanes>(a);
    b = group_sum<kLanes>(b);
  } else {
    block_sums<kLanes>(a, b, shared);
  }
}

// Given what is left of the mean and the mean square of values centred by all but
// that: whether so much is left that the difference of squares would cancel, and the
// values have to be centred anew.
__device__ __forceinline__ bool far_off(float left, float square) { return 64.0f * left * left > square; }

// (A row with an infinity keeps its infinite mean.)
__device__ __forceinline__ float finite_or_zero(float v) { return fabsf(v) < INFINITY ? v : 0.0f; }

// A lane's columns of a row: kPacks times kSize, a pack or, in rows narrower than
// a pack, one.  The last pack of a row that is no whole number of packs begins
// early, so that it ends with the row, and lanes beyond the row take that too:
// what a lane shares with the one before it counts in no sum, and both store the
// same values.
template <int kLanes, int kPacks, int kSize>
struct Columns {
  int64_t at[kPacks];
  int shared_with[kPacks];  // the first values, another lane's
  __device__ __forceinline__ Columns(int lane, int64_t dim) {
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      const int64_t nominal = (int64_t)(k * kLanes + lane) * kSize;
      at[k] = nominal < dim - kSize ? nominal : dim - kSize;
      const int64_t common = nominal - at[k];
      shared_with[k] = common < kSize ? (int)common : kSize;
    }
  }
  // v, or 0 where it counts for another lane.
  __device__ __forceinline__ float own(int k, int e, float v) const { return e >= shared_with[k] ? v : 0.0f; }
  __device__ __forceinline__ bool any(int k) const { return shared_with[k] < kSize; }
};

template <typename W, int kSize>
__device__ __forceinline__ void load_row_part(const W* from, float* out) {
  W w[kSize];
  __builtin_memcpy(w, from, sizeof(w));
#pragma unroll
  for (int e = 0; e < kSize; ++e) out[e] = (float)w[e];
}

template <typename T, typename W, int kLanes, int kPacks, int kSize>
__global__ __launch_bounds__(kLanes > kNormThreads ? kLanes : kNormThreads) void k_norm(
    T* __restrict__ y, float* __restrict__ means, float* __restrict__ rstds, const T* __restrict__ x,
    const W* __restrict__ weight, const W* __restrict__ bias, int64_t rows, int64_t dim, int64_t stride, float eps) {
  constexpr int kThreads = kLanes > kNormThreads ? kLanes : kNormThreads;
  __shared__ float shared[2 * kThreads / kWave];
  const int lane = threadIdx.x % kLanes;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  // Lanes of a row beyond the last only occur where a row is at most a wave's:
  // no barrier follows.
  if (row >= rows) return;
  const Columns<kLanes, kPacks, kSize> columns(lane, dim);
  const T* in = x + row * stride;
  Raw<T, kSize> raw[kPacks];
#pragma unroll
  for (int k = 0; k < kPacks; ++k) raw[k].load(in + columns.at[k]);
  float v[kPacks][kSize];
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < kPacks; ++k) {
    raw[k].get(v[k]);
#pragma unroll
    for (int e = 0; e < kSize; ++e) sum += columns.own(k, e, v[k][e]);
  }
  float mean = row_sum<kLanes>(sum, shared) / (float)dim;
  float left = 0.0f, variance = 0.0f;  // sums of the centred values and of their squares
#pragma unroll
  for (int k = 0; k < kPacks; ++k)
#pragma unroll
    for (int e = 0; e < kSize; ++e) {
      v[k][e] -= mean;
      const float own = columns.own(k, e, v[k][e]);
      left += own;
      variance = fmaf(own, own, variance);
    }
  row_sums<kLanes>(left, variance, shared);
  left = finite_or_zero(left / (float)dim);
  variance /= (float)dim;
  mean += left;
  if (far_off(left, variance)) {  // the same for all lanes of a row
    variance = 0.0f;
#pragma unroll
    for (int k = 0; k < kPacks; ++k)
#pragma unroll
      for (int e = 0; e < kSize; ++e) {
        const float own = columns.own(k, e, v[k][e] - left);
        variance = fmaf(own, own, variance);
      }
    variance = row_sum<kLanes>(variance, shared) / (float)dim;
  } else {
    variance = fmaf(-left, left, variance);
  }
  const float rstd = 1.0f / sqrtf(variance + eps), shift = -left * rstd;
  if (lane == 0) {
    means[row] = mean;
    rstds[row] = rstd;
  }
  T* out = y + row * dim;
#pragma unroll
  for (int k = 0; k < kPacks; ++k) {
    float w[kSize], b[kSize];
    if (weight) load_row_part<W, kSize>(weight + columns.at[k], w);
    if (bias) load_row_part<W, kSize>(bias + columns.at[k], b);
#pragma unroll
    for (int e = 0; e < kSize; ++e) {
      const float h = fmaf(v[k][e], rstd, shift);
      v[k][e] = weight ? (bias ? fmaf(h, w[e], b[e]) : h * w[e]) : h;
    }
    if (columns.any(k)) raw[k].put(v[k], out + columns.at[k]);
  }
}

// Rows wider than the registers of 1024 lanes: three readings, the later two
// from cache (four where the first mean is far off).
template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_norm_wide(T* __restrict__ y, float* __restrict__ means,
                                                    float* __restrict__ rstds, const T* __restrict__ x,
                                                    const W* __restrict__ weight, const W* __restrict__ bias,
                                                    int64_t dim, int64_t stride, float eps) {
  constexpr int kSize = Pack<T>::kSize;
  __shared__ float shared[2 * 1024 / kWave];
  const int64_t row = blockIdx.x;
  const T* in = x + row * stride;
  float v[kSize], w[kSize], b[kSize];
  float sum = 0.0f, left = 0.0f, variance = 0.0f;
  for (int64_t at = (int64_t)threadIdx.x * kSize; at < dim; at += 1024 * kSize) {
    load_pack(in, at, dim, v);
    for (int e = 0; e < kSize; ++e) sum += v[e];
  }
  const float first = block_sum<1024>(sum, shared) / (float)dim;
  for (int64_t at = (int64_t)threadIdx.x * kSize; at < dim; at += 1024 * kSize) {
    load_pack(in, at, dim, v);
    for (int e = 0; e < kSize; ++e) {
      const float c = at + e < dim ? v[e] - first : 0.0f;
      left += c;
      variance = fmaf(c, c, variance);
    }
  }
  block_sums<1024>(left, variance, shared);
  left = finite_or_zero(left / (float)dim);
  variance /= (float)dim;
  const float mean = first + left;
  if (far_off(left, variance)) {  // the same for all lanes
    variance = 0.0f;
    for (int64_t at = (int64_t)threadIdx.x * kSize; at < dim; at += 1024 * kSize) {
      load_pack(in, at, dim, v);
      for (int e = 0; e < kSize; ++e) {
        const float c = at + e < dim ? (v[e] - first) - left : 0.0f;
        variance = fmaf(c, c, variance);
      }
    }
    variance = block_sum<1024>(variance, shared) / (float)dim;
  } else {
    variance = fmaf(-left, left, variance);
  }
  const float rstd = 1.0f / sqrtf(variance + eps);
  if (threadIdx.x == 0) {
    means[row] = mean;
    rstds[row] = rstd;
  }
  for (int64_t at = (int64_t)threadIdx.x * kSize; at < dim; at += 1024 * kSize) {
    load_pack(in, at, dim, v);
    if (weight) load_some<kSize>(weight, at, dim, w);
    if (bias) load_some<kSize>(bias, at, dim, b);
    for (int e = 0; e < kSize; ++e) {
      const float h = ((v[e] - first) - left) * rstd;
      v[e] = weight ? (bias ? fmaf(h, w[e], b[e]) : h * w[e]) : h;
    }
    store_pack(y + row * dim, at, dim, v);
  }
}

// dx row by row; the rows of a workgroup are its column sums' slice, kept in
// registers (a lane holds the same columns of every row) and joined over the
// workgroup's row groups at the end.  The next row is on its way while a row's sums
// cross the lanes.  partial: [workgroup][2][dim], dw then db; one workgroup alone
// has the sums and stores them.
template <typename T, typename W, int kLanes, int kPacks, int kSize>
__global__ __launch_bounds__(gradient_threads(kLanes)) void k_norm_gradient(
    T* __restrict__ dx, float* __restrict__ partial, W* __restrict__ dweight, W* __restrict__ dbias,
    const T* __restrict__ grad, const T* __restrict__ x, const float* __restrict__ means,
    const float* __restrict__ rstds, const W* __restrict__ weight, int64_t rows, int64_t dim, int64_t grad_stride,
    int64_t stride) {
  constexpr int kThreads = gradient_threads(kLanes);
  constexpr int kGroups = kThreads / kLanes;
  __shared__ float shared[kThreads / kWave];
  __shared__ float joined[kGroups > 1 ? kThreads / kWave * kLanes * kSize : 1];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const Columns<kLanes, kPacks, kSize> columns(lane, dim);
  float dw[kPacks][kSize] = {}, db[kPacks][kSize] = {}, w[kPacks][kSize];
#pragma unroll
  for (int k = 0; k < kPacks; ++k)
    if (weight) load_row_part<W, kSize>(weight + columns.at[k], w[k]);
  const float inverse = 1.0f / (float)dim;
  const int64_t step = (int64_t)gridDim.x * kGroups;
  Raw<T, kSize> next_x[kPacks], next_g[kPacks];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int64_t row) {
    if (row >= rows) return;
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      next_x[k].load(x + row * stride + columns.at[k]);
      next_g[k].load(grad + row * grad_stride + columns.at[k]);
    }
    next_mean = means[row];
    next_rstd = rstds[row];
  };
  int64_t row = (int64_t)blockIdx.x * kGroups + group;
  fetch(row);
  // Where a row takes the whole workgroup, all its lanes run the same rows.
  for (; row < rows; row += step) {
    float h[kPacks][kSize], g[kPacks][kSize];
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      next_x[k].get(h[k]);
      next_g[k].get(g[k]);
    }
    const float mean = next_mean, rstd = next_rstd;
    fetch(row + step);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < kPacks; ++k)
#pragma unroll
      for (int e = 0; e < kSize; ++e) {
        h[k][e] = (h[k][e] - mean) * rstd;
        dw[k][e] = fmaf(g[k][e], h[k][e], dw[k][e]);
        db[k][e] += g[k][e];
        if (weight) g[k][e] *= w[k][e];
        const float own = columns.own(k, e, g[k][e]);
        s1 += own;
        s2 = fmaf(own, columns.own(k, e, h[k][e]), s2);
      }
    s1 = row_sum<kLanes>(s1, shared) * inverse;
    s2 = row_sum<kLanes>(s2, shared) * inverse;
    T* out = dx + row * dim;
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
#pragma unroll
      for (int e = 0; e < kSize; ++e) g[k][e] = rstd * (g[k][e] - fmaf(h[k][e], s2, s1));
      if (columns.any(k)) Raw<T, kSize>().put(g[k], out + columns.at[k]);
    }
  }
  if (!partial) return;
  float* slice = partial + (int64_t)blockIdx.x * 2 * dim;
#pragma unroll
  for (int part = 0; part < 2; ++part)
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
      float* mine = part ? db[k] : dw[k];
      if constexpr (kGroups > 1) {
        // The groups of a wave by exchanges, then the waves through LDS.
#pragma unroll
        for (int d = kLanes; d < kWave; d *= 2)
#pragma unroll
          for (int e = 0; e < kSize; ++e) mine[e] += __shfl_xor(mine[e], d, kWave);
        __syncthreads();
        if (threadIdx.x % kWave < kLanes)
#pragma unroll
          for (int e = 0; e < kSize; ++e) joined[(threadIdx.x / kWave * kLanes + lane) * kSize + e] = mine[e];
        __syncthreads();
        if (group) continue;
#pragma unroll
        for (int other = 1; other < kThreads / kWave; ++other)
#pragma unroll
          for (int e = 0; e < kSize; ++e) mine[e] += joined[(other * kLanes + lane) * kSize + e];
      }
      if (!columns.any(k)) continue;
      if (gridDim.x > 1) {
#pragma unroll
        for (int e = 0; e < kSize; ++e) slice[part * dim + columns.at[k] + e] = mine[e];
      } else if (W* to = part ? dbias : dweight) {
#pragma unroll
        for (int e = 0; e < kSize; ++e) to[columns.at[k] + e] = (W)mine[e];
      }
    }
}

// The wide form: a workgroup per strip of rows, as above, with dx in two
// readings and the column sums added up in its slice of `partial`, which only
// this workgroup touches.
template <typename T, typename W>
__global__ __launch_bounds__(1024) void k_norm_gradient_wide(T* __restrict__ dx, float* __restrict__ partial,
                                                             const T* __restrict__ grad, const T* __restrict__ x,
                                                             const float* __restrict__ means,
                                                             const float* __restrict__ rstds,
                                                             const W* __restrict__ weight, int64_t rows, int64_t dim,
                                                             int64_t grad_stride, int64_t stride) {
  constexpr int kSize = Pack<T>::kSize;
  __shared__ float shared[1024 / kWave];
  const float inverse = 1.0f / (float)dim;
  float* slice = partial ? partial + (int64_t)blockIdx.x * 2 * dim : nullptr;
  if (slice && blockIdx.x >= rows)
    for (int64_t at = threadIdx.x; at < 2 * dim; at += 1024) slice[at] = 0.0f;
  float h[kSize], g[kSize], w[kSize];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float mean = means[row], rstd = rstds[row];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t at = (int64_t)threadIdx.x * kSize; at < dim; at += 1024 * kSize) {
      load_pack(x + row * stride, at, dim, h);
      load_pack(grad + row * grad_stride, at, dim, g);
      if (weight) load_some<kSize>(weight, at, dim, w);
      for (int e = 0; e < kSize; ++e) {
        if (at + e >= dim) break;
        h[e] = (h[e] - mean) * rstd;
        if (slice) {
          // Columns at .. at + kSize are this lane's in every row.
          const bool first = row == blockIdx.x;
          float* pw = slice + at + e;
          float* pb = pw + dim;
          *pw = fmaf(g[e], h[e], first ? 0.0f : *pw);
          *pb = g[e] + (first ? 0.0f : *pb);
        }
        if (weight) g[e] *= w[e];
        s1 += g[e];
        s2 = fmaf(g[e], h[e], s2);
      }
    }
    s1 = block_sum<1024>(s1, shared) * inverse;
    s2 = block_sum<1024>(s2, shared) * inverse;
    for (int64_t at = (int64_t)threadIdx.x * kSize; at < dim; at += 1024 * kSize) {
      load_pack(x + row * stride, at, dim, h);
      load_pack(grad + row * grad_stride, at, dim, g);
      if (weight) load_some<kSize>(weight, at, dim, w);
      for (int e = 0; e < kSize; ++e) {
        h[e] = (h[e] - mean) * rstd;
        if (weight) g[e] *= w[e];
        g[e] = rstd * (g[e] - fmaf(h[e], s2, s1));
      }
      store_pack(dx + row * dim, at, dim, g);
    }
  }
}

// dw and db from the workgroups' slices, in their order: a column to a lane,
// kReduceSlices lanes share its slices.
template <typename W>
__global__ __launch_bounds__(kReduceColumns* kReduceSlices) void k_norm_reduce(W* __restrict__ dweight,
                                                                               W* __restrict__ dbias,
                                                                               const float* __restrict__ partial,
                                                                               int64_t dim, int slices) {
  __shared__ float sums[kReduceSlices][kReduceColumns + 1];
  const int column = threadIdx.x % kReduceColumns, part = threadIdx.x / kReduceColumns;
  const int64_t at = (int64_t)blockIdx.x * kReduceColumns + column;
  float sum = 0.0f;
  if (at < 2 * dim)
#pragma unroll 8
    for (int s = part; s < slices; s += kReduceSlices) sum += partial[(int64_t)s * 2 * dim + at];
  sums[part][column] = sum;
  __syncthreads();
  if (part == 0 && at < 2 * dim) {
    for (int p = 1; p < kReduceSlices; ++p) sum += sums[p][column];
    if (at < dim) {
      dweight[at] = (W)sum;
    } else if (dbias) {
      dbias[at - dim] = (W)sum;
    }
  }
}

// Lanes and packs for a row: the least of 1 .. 64 lanes with kWaveElements
// each, then a workgroup's 256 and 1024 with kBlockElements.  Returns 0 where
// the wide form takes the row.
struct RowShape {
  int lanes, packs, size;  // size: values of a pack, 1 in rows narrower than one
};

RowShape row_shape(int64_t dim, int pack, int block_elements) {
  if (dim < pack) return {8, 1, 1};
  const int64_t packs = (dim + pack - 1) / pack;
  int lanes = 1;
  while (lanes < 64 && lanes < packs) lanes *= 2;
  if (lanes == 64 && packs > 64 * (kWaveElements / pack)) lanes = 256;
  if (lanes == 256 && packs > 256 * (kBlockElements / pack)) lanes = 1024;
  if (lanes == 1024 && packs > 1024 * (block_elements / pack)) return {0, 0, pack};
  int each = 1;
  while ((int64_t)each * lanes < packs) each *= 2;
  return {lanes, each, pack};
}

// Calls fn(lanes, packs) with both as constants; the combinations row_shape gives.
template <int kMaxPacks, typename F>
bool with_packs(int packs, F&& fn) {
  switch (packs) {
    case 1: fn(std::integral_constant<int, 1>()); return true;
    case 2: if constexpr (kMaxPacks >= 2) { fn(std::integral_constant<int, 2>()); return true; } break;
    case 4: if constexpr (kMaxPacks >= 4) { fn(std::integral_constant<int, 4>()); return true; } break;
    case 8: if constexpr (kMaxPacks >= 8) { fn(std::integral_constant<int, 8>()); return true; } break;
  }
  return false;
}

template <int kSize, int kWideElements, typename F>
bool with_shape(RowShape shape, F&& fn) {
  using Size = std::integral_constant<int, kSize>;
  using One = std::integral_constant<int, 1>;
  auto lanes = [&](auto l) { return [&, l](auto p) { fn(l, p, Size()); }; };
  if (shape.size == 1) {
    fn(std::integral_constant<int, 8>(), One(), One());
    return true;
  }
  switch (shape.lanes) {
    case 1: return with_packs<1>(shape.packs, lanes(std::integral_constant<int, 1>()));
    case 2: return with_packs<1>(shape.packs, lanes(std::integral_constant<int, 2>()));
    case 4: return with_packs<1>(shape.packs, lanes(std::integral_constant<int, 4>()));
    case 8: return with_packs<1>(shape.packs, lanes(std::integral_constant<int, 8>()));
    case 16: return with_packs<1>(shape.packs, lanes(std::integral_constant<int, 16>()));
    case 32: return with_packs<1>(shape.packs, lanes(std::integral_constant<int, 32>()));
    case 64: return with_packs<kWaveElements / kSize>(shape.packs, lanes(std::integral_constant<int, 64>()));
    case 256: return with_packs<kBlockElements / kSize>(shape.packs, lanes(std::integral_constant<int, 256>()));
    case 1024: return with_packs<kWideElements / kSize>(shape.packs, lanes(std::integral_constant<int, 1024>()));
  }
  return false;
}

template <typename T, typename W>
int norm(T* y, float* mean, float* rstd, const T* x, const W* weight, const W* bias, int64_t rows, int64_t dim,
         int64_t stride, float eps, hipStream_t stream) {
  constexpr int kPack = Pack<T>::kSize;
  const RowShape shape = row_shape(dim, kPack, kBlockElements);
  // A launch holds fewer than 2^32 lanes: very many narrow rows take several.
  constexpr int64_t kRowsAtOnce = int64_t(1) << 21;
  for (int64_t first = 0; first < rows; first += kRowsAtOnce) {
    const int64_t count = rows - first < kRowsAtOnce ? rows - first : kRowsAtOnce;
    const T* in = x + first * stride;
    T* out = y + first * dim;
    const bool done = with_shape<kPack, kBlockElements>(shape, [&](auto l, auto p, auto z) {
      constexpr int kLanes = decltype(l)::value, kPacks = decltype(p)::value, kSize = decltype(z)::value;
      constexpr int kThreads = kLanes > kNormThreads ? kLanes : kNormThreads;
      const uint32_t grid = (uint32_t)((count + kThreads / kLanes - 1) / (kThreads / kLanes));
      hipLaunchKernelGGL((k_norm<T, W, kLanes, kPacks, kSize>), dim3(grid), dim3(kThreads), 0, stream, out, mean + first,
                         rstd + first, in, weight, bias, count, dim, stride, eps);
    });
    if (!done)
      hipLaunchKernelGGL((k_norm_wide<T, W>), dim3((uint32_t)count), dim3(1024), 0, stream, out, mean + first,
                         rstd + first, in, weight, bias, dim, stride, eps);
    MGB_LAUNCH_CHECK("layer norm");
  }
  return 0;
}

// Gradient: 1024 lanes hold half as much of a row, for the column sums.
constexpr int kGradientWideElements = 16;
// One workgroup of 512 to a CU (two of 256), and more rows by turns: their slices
// of the column sums stay small against the rows.  us with half as many, these and
// twice as many: 5,003 x 1,000 binary32 15.6, 13.6, 17.1; 65,536 x 1,024 133, 104, 104;
// 65,536 x 128 25.3, 17.7, 16.7; 8,192 x 4,096 (two of 256) 53.4, 52.9, 60.1.
constexpr int64_t kGradientGroups = 256;

int64_t gradient_slices(int64_t rows, int64_t dim, int size) {
  const RowShape shape = row_shape(dim, size, kGradientWideElements);
  const int64_t at_once = shape.lanes ? gradient_threads(shape.lanes) / shape.lanes : 1;
  const int64_t wanted = (rows + at_once - 1) / at_once, most = shape.lanes == 256 ? 2 * kGradientGroups : kGradientGroups;
  // Two turns of one workgroup cost less than the launch that joins two (9 x 1,000:
  // 5.2 us and 6.9).
  return wanted <= 2 ? 1 : wanted < most ? wanted : most;
}

template <typename T, typename W>
int norm_gradient(T* dx, W* dweight, W* dbias, const T* grad, const T* x, const float* mean, const float* rstd,
                  const W* weight, int64_t rows, int64_t dim, int64_t grad_stride, int64_t stride, float* partial,
                  hipStream_t stream) {
  constexpr int kPack = Pack<T>::kSize;
  const RowShape shape = row_shape(dim, kPack, kGradientWideElements);
  const int64_t slices = gradient_slices(rows, dim, kPack);
  if (!dweight) partial = nullptr;
  if (rows || partial) {
    const bool done = with_shape<kPack, kGradientWideElements>(shape, [&](auto l, auto p, auto z) {
      constexpr int kLanes = decltype(l)::value, kPacks = decltype(p)::value, kSize = decltype(z)::value;
      constexpr int kThreads = gradient_threads(kLanes);
      hipLaunchKernelGGL((k_norm_gradient<T, W, kLanes, kPacks, kSize>), dim3((uint32_t)slices), dim3(kThreads), 0,
                         stream, dx, partial, dweight, dbias, grad, x, mean, rstd, weight, rows, dim, grad_stride, stride);
    });
    if (!done)
      hipLaunchKernelGGL((k_norm_gradient_wide<T, W>), dim3((uint32_t)slices), dim3(1024), 0, stream, dx, partial, grad,
                         x, mean, rstd, weight, rows, dim, grad_stride, stride);
    MGB_LAUNCH_CHECK("layer norm gradient");
    if (done && slices == 1) partial = nullptr;
  }
  if (partial) {
    hipLaunchKernelGGL((k_norm_reduce<W>), dim3((uint32_t)((2 * dim + kReduceColumns - 1) / kReduceColumns)),
                       dim3(kReduceColumns * kReduceSlices), 0, stream, dweight, dbias, partial, dim, (int)slices);
    MGB_LAUNCH_CHECK("layer norm parameter gradients");
  }
  return 0;
}

// fn(data type, parameter type): parameters are binary32 or the data's type.
template <typename F>
int with_types(int dtype, int weight_dtype, F&& fn) {
  if (dtype == MGB_F32 && weight_dtype == MGB_F32) return fn((float*)nullptr, (float*)nullptr);
  if (dtype == MGB_F16 && weight_dtype == MGB_F16) return fn((_Float16*)nullptr, (_Float16*)nullptr);
  if (dtype == MGB_F16 && weight_dtype == MGB_F32) return fn((_Float16*)nullptr, (float*)nullptr);
  if (dtype == MGB_BF16 && weight_dtype == MGB_BF16) return fn((__bf16*)nullptr, (__bf16*)nullptr);
  if (dtype == MGB_BF16 && weight_dtype == MGB_F32) return fn((__bf16*)nullptr, (float*)nullptr);
  set_error("layer norm: types must be float32, float16 or bfloat16, parameters float32 or the data's type");
  return -1;
}

int check_rows(int64_t rows, int64_t dim, int64_t stride) {
  MGB_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31), "layer norm: rows must be below 2^31");
  MGB_REQUIRE(dim >= 1 && dim < (int64_t(1) << 31), "layer norm: a row must have 1 to 2^31 - 1 values");
  // Row strides of either sign and of 0 (a broadcast row) are addresses like others.
  MGB_REQUIRE(stride < (int64_t(1) << 40) && stride > -(int64_t(1) << 40), "layer norm: row stride out of range");
  return 0;
}

}  // namespace
}  // namespace mgb

using namespace mgb;

extern "C" {

int mgb_layer_norm(void* y, float* mean, float* rstd, const void* x, const void* weight, const void* bias, int64_t rows,
                   int64_t dim, int64_t stride, float eps, int dtype, int weight_dtype, void* stream) {
  if (check_rows(rows, dim, stride)) return -1;
  MGB_REQUIRE(weight || !bias, "layer norm: a bias needs a weight");
  if (rows == 0) return 0;
  MGB_REQUIRE(y && mean && rstd && x, "layer norm: null pointer");
  return with_types(dtype, weight_dtype, [&](auto* t, auto* w) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    return norm<T, W>((T*)y, mean, rstd, (const T*)x, (const W*)weight, (const W*)bias, rows, dim, stride, eps,
                      (hipStream_t)stream);
  });
}

size_t mgb_layer_norm_gradient_workspace_bytes(int64_t rows, int64_t dim, int dtype) {
  if (rows < 0 || dim < 1) return 0;
  return (size_t)gradient_slices(rows, dim, dtype == MGB_F32 ? 4 : 8) * 2 * dim * sizeof(float);
}

int mgb_layer_norm_gradient(void* dx, void* dweight, void* dbias, const void* grad, const void* x, const float* mean,
                            const float* rstd, const void* weight, int64_t rows, int64_t dim, int64_t grad_stride,
                            int64_t stride, int dtype, int weight_dtype, void* workspace, size_t workspace_bytes,
                            void* stream) {
  if (check_rows(rows, dim, stride) || check_rows(rows, dim, grad_stride)) return -1;
  MGB_REQUIRE(dweight || !dbias, "layer norm gradient: a bias' gradient needs the weight's");
  MGB_REQUIRE(!dweight || workspace_bytes >= mgb_layer_norm_gradient_workspace_bytes(rows, dim, dtype),
              "layer norm gradient: workspace too small");
  MGB_REQUIRE(!dweight || workspace, "layer norm gradient: null workspace");
  MGB_REQUIRE(rows == 0 || (dx && grad && x && mean && rstd), "layer norm gradient: null pointer");
  return with_types(dtype, weight_dtype, [&](auto* t, auto* w) {
    using T = std::remove_pointer_t<decltype(t)>;
    using W = std::remove_pointer_t<decltype(w)>;
    return norm_gradient<T, W>((T*)dx, (W*)dweight, (W*)dbias, (const T*)grad, (const T*)x, mean, rstd,
                               (const W*)weight, rows, dim, grad_stride, stride, (float*)workspace,
                               (hipStream_t)stream);
  });
}

}  // extern "C"
