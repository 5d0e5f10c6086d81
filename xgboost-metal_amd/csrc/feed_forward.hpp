// What the block's forward and backward passes share (feed_forward.hip,
// feed_forward_gradient.hip): the operands' layout, the plan of a product, the
// activations.
#pragma once
#include <algorithm>
#include <vector>

#include "product_parts.hpp"

namespace mgb {
namespace block {

using product::Params;
using product::float4v;

// (Rows: as many as tiles of 256 by 512 lanes take in a launch, which holds fewer than 2^32.)
constexpr int64_t kMostSide = int64_t(1) << 20, kMostRows = (int64_t(1) << 31) - 2048;

// The matrix instructions' type for values of T, and the parts that hold one.
// Binary32 values are three bfloat16, 24 bits (or 2^-134, where bfloat16's steps end),
// whose products take six instructions; the type has binary32's range, so nothing is
// scaled.
template <typename T>
struct Kind {
  using E = T;
  static constexpr int kParts = 1, kPairs = 1;
};
template <>
struct Kind<float> {
  using E = __bf16;
  static constexpr int kParts = 3, kPairs = 6;
};

// v as the sum of three bfloat16.  What is not finite stays as it is in the first;
// a value that would round to an infinity is cut instead.
__device__ __forceinline__ void split_parts(float v, __bf16* part) {
  __bf16 first = (__bf16)v;
  if (!(fabsf((float)first) < INFINITY)) {
    const uint32_t cut = __float_as_uint(v) & 0xffff0000u;
    if (fabsf(v) < INFINITY) first = (__bf16)__uint_as_float(cut);
  }
  float rest = v - (float)first;
  if (!(fabsf(rest) < INFINITY)) rest = 0.0f;
  part[0] = first;
  part[1] = (__bf16)rest;
  part[2] = (__bf16)(rest - (float)part[1]);
}

// Workspace in pieces; without a base it counts.
struct Space {
  char* base;
  size_t used;
  char* take(size_t bytes) {
    char* at = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return at;
  }
};

// Rows of the inner matrices: those of whole 2 KB would all begin in the same few
// of the cache's channels (products of 8,192 x 8,192 x 8,192: 862 us, and 770 with rows
// of 1 KB more), so they are 256 bytes longer.
inline int64_t inner_stride(int64_t columns) { return columns % 1024 ? columns : columns + 128; }

// ---- layout ------------------------------------------------------------------
// The products load 16 bytes a lane, whole ones of a row.  16-bit matrices whose
// rows begin at 16 bytes and hold whole ones are read where they lie; others are
// copied with their rows padded with zeros, and binary32 ones split into parts.
struct LayJob {
  const void* from;
  char* to;
  int64_t rows, columns, stride, chunks, part;  // stride in elements, chunks of 8 a row of `to`, part in bytes
  bool turned;
};
constexpr int kMostLay = 5;
struct LayJobs {
  LayJob job[kMostLay];
  int count;
};

constexpr int kLayThreads = 256;

template <typename T>
__device__ __forceinline__ void lay_straight(const LayJob& job) {
  using E = typename Kind<T>::E;
  constexpr int kParts = Kind<T>::kParts;
  const int64_t all = job.rows * job.chunks, step = (int64_t)gridDim.x * kLayThreads;
  const int64_t step_rows = step / job.chunks, step_chunks = step % job.chunks;
  int64_t at = (int64_t)blockIdx.x * kLayThreads + threadIdx.x, row = at / job.chunks, chunk = at % job.chunks;
  for (; at < all; at += step) {
    float v[8];
    load_some<8>((const T*)job.from + row * job.stride, chunk * 8, job.columns, v);
    E part[kParts][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (kParts == 3) {
        __bf16 three[3];
        split_parts(v[e], three);
#pragma unroll
        for (int q = 0; q < 3; ++q) part[q][e] = three[q];
      } else {
        part[0][e] = (E)v[e];
      }
    }
#pragma unroll
    for (int q = 0; q < kParts; ++q)
      __builtin_memcpy(__builtin_assume_aligned(job.to + q * job.part + (row * job.chunks + chunk) * 16, 16), part[q], 16);
    row += step_rows;
    chunk += step_chunks;
    if (chunk >= job.chunks) {
      chunk -= job.chunks;
      ++row;
    }
  }
}

// The same, transposed: rows of `to` are columns of `from`.
constexpr int kTurnSide = 64;
template <typename T>
__device__ __forceinline__ void lay_across(const LayJob& job) {
  using E = typename Kind<T>::E;
  constexpr int kParts = Kind<T>::kParts;
  __shared__ float tile[kTurnSide][kTurnSide + 1];
  const int64_t across = (job.columns + kTurnSide - 1) / kTurnSide, down = (job.rows + kTurnSide - 1) / kTurnSide;
  for (int64_t at = blockIdx.x; at < across * down; at += gridDim.x) {
    const int64_t row0 = at / across * kTurnSide, column0 = at % across * kTurnSide;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTurnSide * kTurnSide / 8 / kLayThreads; ++k) {
      const int eight = k * kLayThreads + threadIdx.x, row = eight / (kTurnSide / 8), column = eight % (kTurnSide / 8) * 8;
      float v[8] = {};
      if (row0 + row < job.rows) load_some<8>((const T*)job.from + (row0 + row) * job.stride, column0 + column, job.columns, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) tile[row][column + e] = v[e];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTurnSide * kTurnSide / 8 / kLayThreads; ++k) {
      // (lanes that follow each other take rows of `to`: columns of the tile lie in different banks)
      const int eight = k * kLayThreads + threadIdx.x, row = eight % kTurnSide, chunk = eight / kTurnSide;
      if (column0 + row >= job.columns || row0 / 8 + chunk >= job.chunks) continue;
      E part[kParts][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = tile[chunk * 8 + e][row];
        if constexpr (kParts == 3) {
          __bf16 three[3];
          split_parts(v, three);
#pragma unroll
          for (int q = 0; q < 3; ++q) part[q][e] = three[q];
        } else {
          part[0][e] = (E)v;
        }
      }
#pragma unroll
      for (int q = 0; q < kParts; ++q)
        __builtin_memcpy(__builtin_assume_aligned(job.to + q * job.part + ((column0 + row) * job.chunks + row0 / 8 + chunk) * 16, 16),
                         part[q], 16);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kLayThreads) void k_lay_out(LayJobs jobs) {
  const LayJob& job = jobs.job[blockIdx.y];
  if (job.turned) lay_across<T>(job);
  else lay_straight<T>(job);
}

// A matrix as a product takes it.
struct Laid {
  const char* data;
  int64_t stride, part;  // bytes
};

inline int64_t padded(int64_t n) { return (n + 7) / 8 * 8; }

template <typename T>
bool lies_well(const void* data, int64_t rows, int64_t columns, int64_t stride) {
  return sizeof(T) == 2 && columns % 8 == 0 && (uintptr_t)data % 16 == 0 &&
         (rows <= 1 || (stride % 8 == 0 && stride >= columns && stride <= kMostSide));
}

template <typename T>
Laid lay(Space& space, LayJobs& jobs, const void* data, int64_t rows, int64_t columns, int64_t stride, bool copy) {
  if (!copy) return {(const char*)data, (rows > 1 ? stride : columns) * 2, 0};
  const int64_t width = padded(columns) * 2, part = width * rows;
  char* to = space.take(part * Kind<T>::kParts);
  jobs.job[jobs.count++] = {data, to, rows, columns, stride, width / 16, part, false};
  return {to, width, part};
}

template <typename T>
Laid lay(Space& space, LayJobs& jobs, const void* data, int64_t rows, int64_t columns, int64_t stride) {
  return lay<T>(space, jobs, data, rows, columns, stride, !lies_well<T>(data, rows, columns, stride));
}

// The transpose (columns, rows) of a matrix.
template <typename T>
Laid lay_turned(Space& space, LayJobs& jobs, const void* data, int64_t rows, int64_t columns, int64_t stride) {
  const int64_t width = inner_stride(padded(rows)) * 2, part = width * columns;
  char* to = space.take(part * Kind<T>::kParts);
  jobs.job[jobs.count++] = {data, to, rows, columns, stride, width / 16, part, true};
  return {to, width, part};
}

template <typename T>
void lay_out(const LayJobs& jobs, hipStream_t stream) {
  int64_t most = 0;
  for (int k = 0; k < jobs.count; ++k) {
    const LayJob& job = jobs.job[k];
    most = std::max(most, job.turned ? ((job.rows + kTurnSide - 1) / kTurnSide) * ((job.columns + kTurnSide - 1) / kTurnSide)
                                     : (job.rows * job.chunks + kLayThreads - 1) / kLayThreads);
  }
  if (most == 0) return;
  const int64_t groups = std::min<int64_t>(most, 4096);
  k_lay_out<T><<<dim3((uint32_t)groups, jobs.count), kLayThreads, 0, stream>>>(jobs);
}

// A 16-bit result's own rounding and that of the inner values add up to 1.41 times one of
// them, of many values; among few there are some where it is twice.  Blocks with so few
// results (or a gradient of a matrix) keep what the inner values' rounding leaves as well
// and add its products, which costs them little: 33 x 248 x 1,024 in bfloat16 13.4 us,
// its gradients 25.4; without 12.3 and 20.9.
constexpr int64_t kFewResults = 8192;

// ---- a product's plan ----------------------------------------------------------
enum Size { kLarge, kMedium, kSmall };
inline int side(Size size) { return size == kLarge ? 256 : size == kMedium ? 128 : 64; }

inline uint32_t lay_tiles(Params& p, Size size, bool dual) {
  const int64_t m = side(size), n = dual ? m / 2 : m;
  p.tiles = 0;
  for (int j = 0; j < p.jobs; ++j) {
    auto& job = p.job[j];
    job.first_tile = p.tiles;
    job.row_tiles = (uint32_t)((job.rows + m - 1) / m);
    job.column_tiles = (uint32_t)((job.columns + n - 1) / n);
    p.tiles += job.row_tiles * job.column_tiles;
  }
  return p.tiles;
}

// Steps of a workgroup that has the whole depth.  Parts' products go by k_product's
// large tiles, or by k_parts' smaller ones, which have all six in a step of 32.
inline bool in_parts(const Params& p, Size size) { return p.pairs > 1 && size != kLarge; }
inline int64_t steps_of(const Params& p, Size size, int values) {
  const bool parts = in_parts(p, size);
  if (parts) values = 32;
  return std::max<int64_t>(1, (p.depth + values - 1) / values) * (parts ? 1 : p.pairs) * p.sources;
}

// Estimated times, in us, of a workgroup's step and of what comes before and after its
// steps, with 1, 2, .. workgroups a compute unit (measured with 64 to 1,024 tiles and
// depths of 512 to 4,096; turned operands' steps take a third longer, of k_parts a
// twelfth).  Products of few tiles are short of workgroups, those of many small ones of
// LDS' rate: the estimate finds sizes and shares between.
struct Rate {
  int most;       // workgroups a compute unit
  float step[4], fixed[4];
};
constexpr Rate kRates[3] = {{1, {1.42f}, {10.0f}},
                            {2, {0.575f, 0.87f}, {6.4f, 8.8f}},
                            {4, {0.346f, 0.446f, 0.6f, 0.748f}, {4.9f, 5.3f, 6.5f, 7.6f}}};
constexpr Rate kPartRates[3] = {{}, {1, {1.3f}, {8.0f}}, {2, {0.53f, 0.95f}, {7.5f, 7.5f}}};  // of k_parts
constexpr int64_t kUnits = 256;  // compute units

// (Each of the 8 chiplets of 32 units has an eighth of the tiles, find_tile's stretch.)
inline float estimate(const Params& p, Size size, int64_t tiles, int64_t shares, int64_t steps, bool turned) {
  const Rate& r = in_parts(p, size) ? kPartRates[size] : kRates[size];
  const float longer = !turned ? 1.0f : in_parts(p, size) ? 1.08f : 1.3f;
  const int64_t each = ((tiles + 7) / 8 * shares + kUnits / 8 - 1) / (kUnits / 8);
  float time = 0.0f;
  for (int64_t left = each; left > 0;) {  // rounds of r.most, the last of what is left
    const int64_t rounds = left >= r.most ? left / r.most : 1, now = left >= r.most ? r.most : left;
    time += rounds * (r.fixed[now - 1] + steps * r.step[now - 1] * longer);
    left -= rounds * now;
  }
  return time;
}

// Added to the estimates of what no launch holds.  Very many rows of few columns take larger
// tiles than they would otherwise.
inline float too_many(const Params& p, Size size, int64_t tiles, int64_t shares) {
  int64_t lanes = size == kLarge ? product::Large::kThreads : size == kMedium ? product::Medium::kThreads : product::Small::kThreads;
  if (in_parts(p, size)) lanes = size == kMedium ? product::PartMedium::kThreads : product::PartSmall::kThreads;
  return (tiles + 7) / 8 * 8 * shares * lanes < int64_t(1) << 32 ? 0.0f : 1e12f;
}

// The size of the tiles where the depth stays whole.
inline Size choose(Params& p, bool dual, int values = 64) {
  Size best = kSmall;
  float least = INFINITY;
  for (const Size size : {kLarge, kMedium, kSmall}) {
    const int64_t tiles = lay_tiles(p, size, dual);
    const float time = estimate(p, size, tiles, 1, steps_of(p, size, values), false) + too_many(p, size, tiles, 1);
    if (time < least) {
      least = time;
      best = size;
    }
  }
  lay_tiles(p, best, dual);
  p.splits = 1;
  p.first_steps = p.other_steps = (uint32_t)steps_of(p, best, values);
  return best;
}

// The same where the depth may be shared: each tile's shares are workgroups of their own,
// whose partial sums, in binary32, k_join adds in their order.  Shares of one length,
// or, of large tiles that leave compute units idle, a first one as long as the whole
// work is to take and shorter ones for the idle units.
inline Size choose_shares(Params& p, Space& space, bool turned, int values = 64, int64_t most_steps = INT32_MAX) {
  Size best = kSmall;
  int64_t best_first = 0, best_other = 0;
  float least = INFINITY;
  auto consider = [&](Size size, int64_t first, int64_t other, float time) {
    if (time >= least || first > most_steps || other > most_steps) return;
    least = time;
    best = size;
    best_first = first;
    best_other = other;
  };
  for (const Size size : {kLarge, kMedium, kSmall}) {
    const int64_t tiles = lay_tiles(p, size, false), steps = steps_of(p, size, values);
    const float area = (float)side(size) * side(size) * tiles * 8.0f / 5e6f;  // written and read again, 5 TB/s
    // (64 shares of most_steps need not hold the depth: then as many as do, in eights.)
    const int64_t most_shares = std::max<int64_t>(64, ((steps + most_steps - 1) / most_steps + 7) / 8 * 8);
    for (int64_t shares = 1; shares <= most_shares; shares += shares < 8 ? 1 : shares < 16 ? 2 : 8) {
      const int64_t each = (steps + shares - 1) / shares;
      if (shares > 1 && each < 4 && each * (shares - 1) >= steps) break;
      consider(size, each, each, estimate(p, size, tiles, shares, each, turned) + (shares > 1 ? 3.0f + area * shares : 0.0f) +
                                     too_many(p, size, tiles, shares));
    }
    if (size != kLarge || tiles <= kUnits / 2 || tiles >= kUnits) continue;
    const int64_t first = (steps * tiles + kUnits - 1) / kUnits, rest = steps - first;
    for (int64_t shares = 1; shares <= 6 && rest >= shares; ++shares) {
      const int64_t other = (rest + shares - 1) / shares, rounds = (tiles * shares + kUnits - tiles - 1) / (kUnits - tiles);
      const float idle = rounds * estimate(p, size, 1, 1, other, turned), own = estimate(p, size, 1, 1, first, turned);
      consider(size, first, other, std::max(idle, own) + 3.0f + area * (1 + shares));
    }
  }
  lay_tiles(p, best, false);
  const int64_t steps = steps_of(p, best, values);
  p.first_steps = (uint32_t)std::min(best_first, steps);
  p.other_steps = (uint32_t)best_other;
  p.splits = steps > best_first ? 1 + (uint32_t)((steps - best_first + best_other - 1) / best_other) : 1;
  p.partial_size = 0;
  for (int j = 0; j < p.jobs; ++j) {
    p.job[j].partial = p.partial_size;
    p.partial_size += (p.job[j].rows * p.job[j].columns + 3) / 4 * 4;
  }
  p.partials = p.splits > 1 ? (float*)space.take(p.splits * p.partial_size * sizeof(float)) : nullptr;
  return best;
}

template <typename T>
__global__ __launch_bounds__(256) void k_join(Params p) {
  const product::Job& job = p.job[blockIdx.y];
  const int64_t all = job.rows * job.columns, step = (int64_t)gridDim.x * 256 * 4;
  T* out = (T*)job.out;
  for (int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; at < all; at += step) {
    const float* from = p.partials + job.partial + at;
    float4v sum = *(const float4v*)from;
    for (uint32_t s = 1; s < p.splits; ++s) sum += *(const float4v*)(from + s * p.partial_size);
    if (at + 4 <= all) {
      T r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = (T)sum[e];
      __builtin_memcpy(out + at, r, sizeof(r));
    } else {
      for (int e = 0; at + e < all; ++e) out[at + e] = (T)sum[e];
    }
  }
}

// T: the values' type, whose parts k_parts multiplies in smaller tiles.
template <typename E, typename T, bool kLeftTurned, bool kRightTurned, class Finish>
void launch_product(const Params& p, Size size, hipStream_t stream) {
  const uint32_t groups = (p.tiles + 7) / 8 * 8 * p.splits;
  auto launch = [&](auto tile) {
    using S = decltype(tile);
    product::k_product<E, kLeftTurned, kRightTurned, S, Finish><<<groups, S::kThreads, 0, stream>>>(p);
  };
  if (size == kLarge) return launch(product::Large{});
  if constexpr (Kind<T>::kParts == 3) {
    auto parts = [&](auto tile) {
      using S = decltype(tile);
      product::k_parts<kLeftTurned, kRightTurned, S, Finish><<<groups, S::kThreads, 0, stream>>>(p);
    };
    if (size == kMedium) parts(product::PartMedium{});
    else parts(product::PartSmall{});
  } else {
    if (size == kMedium) launch(product::Medium{});
    else launch(product::Small{});
  }
}

// Products whose results are stored as they are, without gaps; Out: their type.
template <typename E, typename T, typename Out, bool kLeftTurned, bool kRightTurned>
void store_product(const Params& p, Size size, hipStream_t stream) {
  if (p.splits == 1) {
    launch_product<E, T, kLeftTurned, kRightTurned, product::Store<Out>>(p, size, stream);
    return;
  }
  launch_product<E, T, kLeftTurned, kRightTurned, product::Partial>(p, size, stream);
  int64_t most = 0;
  for (int j = 0; j < p.jobs; ++j) most = std::max(most, p.job[j].rows * p.job[j].columns);
  k_join<Out><<<dim3((uint32_t)std::min<int64_t>((most + 1023) / 1024, 2048), p.jobs), 256, 0, stream>>>(p);
}

// ---- activations -----------------------------------------------------------------
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float inverse(float v) { return __builtin_amdgcn_rcpf(v); }

// Both of 1 ulp, as is the exponent's rounding times |g|: silu is off by about
// (|g| + 3) 2^-24 of itself.
__device__ __forceinline__ float logistic(float g) { return inverse(1.0f + exp2_fast(g * -1.44269504f)); }

// The normal distribution's function Phi(g), and exp(-g^2 / 2).  For z = |g| / sqrt(2)
// and t = 1 / (1 + c z), Phi(-|g|) = exp(-z^2) t P(t) / 2, with P fitted to
// t^-1 exp(z^2) erfc(z) by least squares, weighted until the relative error is even:
// 7e-6 with six coefficients (16-bit results), 1.1e-8 with nine (binary32 results,
// where the roundings are 4e-7 for g above -12).
template <bool kExact>
__device__ __forceinline__ float normal(float g, float* density) {
  constexpr float kC = kExact ? 0.375f : 0.425f;
  const float e = exp2_fast(g * g * -0.72134752f);
  *density = e;
  const float t = inverse(fmaf(fabsf(g), kC * 0.70710678f, 1.0f));
  float poly;
  if constexpr (kExact) {
    poly = fmaf(t, 0.0616967715f, -0.288076133f);
    poly = fmaf(t, poly, 0.43389535f);
    poly = fmaf(t, poly, -0.231078207f);
    poly = fmaf(t, poly, 0.274845332f);
    poly = fmaf(t, poly, 0.121038452f);
    poly = fmaf(t, poly, 0.205430552f);
    poly = fmaf(t, poly, 0.210633487f);
    poly = fmaf(t, poly, 0.211614415f);
  } else {
    poly = fmaf(t, -0.154950291f, 0.431325078f);
    poly = fmaf(t, poly, -0.0336631872f);
    poly = fmaf(t, poly, 0.288952172f);
    poly = fmaf(t, poly, 0.227761433f);
    poly = fmaf(t, poly, 0.2405819f);
  }
  const float tail = 0.5f * t * poly * e;
  return g < 0.0f ? tail : 1.0f - tail;
}

template <bool kExact>
__device__ __forceinline__ float activate(float g, int activation) {
  if (activation == MGB_SILU) return g * logistic(g);
  float density;
  return g * normal<kExact>(g, &density);
}

// act(g), and its derivative.
template <bool kExact>
__device__ __forceinline__ float activate(float g, int activation, float* slope) {
  if (activation == MGB_SILU) {
    const float s = logistic(g);
    *slope = s * fmaf(g, 1.0f - s, 1.0f);
    return g * s;
  }
  float density;
  const float phi = normal<kExact>(g, &density);
  *slope = fmaf(g * density, 0.39894228f, phi);
  return g * phi;
}

// Values of a row of the block's inner matrices, in parts; kRest: with what the rounding
// of 16-bit ones leaves, from `rest` on.
template <typename T, bool kRest, int kCount>
__device__ __forceinline__ void store_inner(char* matrix, int64_t part, int64_t rest, int64_t at, const float* v) {
  using E = typename Kind<T>::E;
  constexpr int kParts = Kind<T>::kParts;
  E some[kParts][kCount];
#pragma unroll
  for (int e = 0; e < kCount; ++e) {
    if constexpr (kParts == 3) {
      __bf16 three[3];
      split_parts(v[e], three);
#pragma unroll
      for (int q = 0; q < 3; ++q) some[q][e] = three[q];
    } else {
      some[0][e] = (E)v[e];
    }
  }
#pragma unroll
  for (int q = 0; q < kParts; ++q)
    __builtin_memcpy(__builtin_assume_aligned(matrix + (q * part + at) * 2, kCount * 2), some[q], kCount * 2);
  if constexpr (kRest) {
    static_assert(kParts == 1, "parts leave nothing");
#pragma unroll
    for (int e = 0; e < kCount; ++e) {
      const float left = v[e] - (float)some[0][e];
      some[0][e] = (E)(fabsf(left) < INFINITY ? left : 0.0f);
    }
    __builtin_memcpy(__builtin_assume_aligned(matrix + (rest + at) * 2, kCount * 2), some[0], kCount * 2);
  }
}

inline product::Operand operand(const Laid& m, int64_t extent, int64_t depth) {
  return {{m.data, nullptr}, {m.stride, m.stride}, m.part, extent, depth};
}
inline product::Operand operands(const Laid& m, const Laid& second, int64_t extent, int64_t depth) {
  return {{m.data, second.data, m.data, second.data}, {m.stride, second.stride, m.stride, second.stride}, m.part, extent, depth};
}

}  // namespace block
}  // namespace mgb
