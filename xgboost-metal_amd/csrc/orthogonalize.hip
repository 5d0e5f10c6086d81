// A matrix's update made orthogonal by Newton-Schulz products (the Muon
// optimiser's update): with X0 = G / (|G|_F + eps), m x n and m <= n (taller
// ones transposed),
//   X <- (a I + b A + c A^2) X,   A = X X^T,   `steps` times.
// Every step is a polynomial Z in A applied from the left, so a segment of
// steps runs among m x m matrices: A <- Z A Z and P <- Z P, all symmetric and
// commuting, and one product X <- P X ends it.  For n > m that leaves out most
// products with n; symmetric results take half their tiles.  An error in A grows
// by a^2 a step where X is small, so a segment has at most kSegment steps and
// the next one takes A from X anew: with three, the result is as near the
// exact one as binary32 products of the plain form come (low rank 512 x 2048:
// 4e-5 of the norm against 2e-5; all five in one segment: 1e-4).
//
// The matrix instructions multiply binary16.  A small direction's part grows
// a-fold a step, so operands of 11 bits would show in the result (4e-2 of the
// norm at low rank, after five steps): each value is the sum of two binary16
// numbers, 22 bits, and a product takes three matrix instructions (high by
// high, high by low, low by high; low by low is below binary32's rounding).
// Sums are binary32.
#include <utility>

#include "encoder_common.hpp"

namespace mgb {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;      // rows and columns of a workgroup's tile, and the padding of every matrix
constexpr int kDepth = 64;     // depth of a stage in LDS
constexpr int kSegment = 3;
constexpr int kNormGroups = 256;
constexpr int64_t kMostSide = int64_t(1) << 20;
// With these a segment's P stays far below binary16's 65,504 while X's singular
// values are at most about 1.
constexpr float kMostCoefficient = 8.0f;

// Stored values are scaled so that the low part stays a normal number: entries
// of X and A are at most about 1, those of Z and P at most a^kSegment.
constexpr float kScaleX = 4096.0f, kScaleZ = 64.0f;

using half8 = __attribute__((ext_vector_type(8))) _Float16;
using float4v = __attribute__((ext_vector_type(4))) float;

// High and low parts of a matrix, rows of `stride` values.
struct Split {
  _Float16 *high, *low;
  int64_t stride, batch_stride;
};

__device__ __forceinline__ void split_store(const Split& m, int64_t batch, int64_t row, int64_t column, float v) {
  const _Float16 high = (_Float16)v;
  const int64_t at = batch * m.batch_stride + row * m.stride + column;
  m.high[at] = high;
  m.low[at] = (_Float16)(v - (float)high);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void k_square_sums(float* __restrict__ partial, const T* __restrict__ g,
                                                          int64_t rows, int64_t columns, int64_t stride,
                                                          int64_t batch_stride) {
  __shared__ float shared[kThreads / kWave];
  constexpr int kSize = Pack<T>::kSize;
  const T* in = g + blockIdx.y * batch_stride;
  const int64_t packs = (columns + kSize - 1) / kSize, total = rows * packs;
  float sum = 0.0f, v[kSize];
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / packs;
    load_pack(in + row * stride, (i - row * packs) * kSize, columns, v);
#pragma unroll
    for (int e = 0; e < kSize; ++e) sum = fmaf(v[e], v[e], sum);
  }
  sum = block_sum<kThreads>(sum, shared);
  if (threadIdx.x == 0) partial[blockIdx.y * kNormGroups + blockIdx.x] = sum;
}

// G scaled, as it lies and transposed, both with zeros up to whole tiles.
template <typename T>
__global__ __launch_bounds__(kThreads) void k_normalize(Split straight, Split turned, const T* __restrict__ g,
                                                        const float* __restrict__ partial, int64_t rows,
                                                        int64_t columns, int64_t stride, int64_t batch_stride,
                                                        float eps) {
  __shared__ float shared[kThreads / kWave];
  __shared__ float tile[kTile][kTile + 1];
  const int64_t batch = blockIdx.z;
  const float norm = sqrtf(block_sum<kThreads>(partial[batch * kNormGroups + threadIdx.x], shared));
  const float factor = kScaleX / (norm + eps);
  const T* in = g + batch * batch_stride;
  const int64_t row0 = (int64_t)blockIdx.y * kTile, column0 = (int64_t)blockIdx.x * kTile;
  const int x = threadIdx.x % kTile;
  for (int y = threadIdx.x / kTile; y < kTile; y += kThreads / kTile) {
    const float v = row0 + y < rows && column0 + x < columns
                        ? (float)in[(row0 + y) * stride + column0 + x] * factor : 0.0f;
    tile[y][x] = v;
    split_store(straight, batch, row0 + y, column0 + x, v);
  }
  __syncthreads();
  for (int y = threadIdx.x / kTile; y < kTile; y += kThreads / kTile)
    split_store(turned, batch, column0 + y, row0 + x, tile[x][y]);
}

// What a product's tile becomes.
enum { kSymmetric, kBoth, kFinal };

struct Product {
  Split left, right;       // result = left right^T, both with rows of `depth` values
  Split out, turned;       // kSymmetric: out; kBoth: out and its transpose
  Split added;             // kSymmetric with `added.high`: + added_factor added + diagonal I
  int64_t depth;
  float factor, added_factor, diagonal;
  void* result;            // kFinal: the caller's matrix, element (i, j) at i row_step + j column_step
  int64_t rows, columns, row_step, column_step, result_batch;
};

// LDS rows of kDepth binary16 values are 128 bytes, as wide as the banks; the
// 16-byte piece a lane wants of row r lies at piece ^ (r >> 1 & 7), so that 16
// rows' pieces fall on different banks.
__device__ __forceinline__ int piece_at(int row, int piece) {
  return row * (kDepth / 8) + (piece ^ (row >> 1 & 7));
}

template <int kMode, typename T>
__global__ __launch_bounds__(kThreads) void k_product(Product p) {
  __shared__ half8 lds[4][kTile * kDepth / 8];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t batch = blockIdx.z;
  int64_t ti = blockIdx.y, tj = blockIdx.x;
  if constexpr (kMode == kSymmetric) {
    // Tiles on and above the diagonal, counted column by column.
    const uint32_t t = blockIdx.x;
    uint32_t j = (uint32_t)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while (j * (j + 1) / 2 > t) --j;
    while ((j + 1) * (j + 2) / 2 <= t) ++j;
    tj = j;
    ti = t - j * (j + 1) / 2;
  }
  const _Float16* from[4] = {
      p.left.high + batch * p.left.batch_stride + ti * kTile * p.left.stride,
      p.left.low + batch * p.left.batch_stride + ti * kTile * p.left.stride,
      p.right.high + batch * p.right.batch_stride + tj * kTile * p.right.stride,
      p.right.low + batch * p.right.batch_stride + tj * kTile * p.right.stride};
  const int64_t stride[4] = {p.left.stride, p.left.stride, p.right.stride, p.right.stride};
  constexpr int kPieces = kTile * kDepth / 8 / kThreads;  // of each of the four, a lane's
  half8 held[4][kPieces];
  auto fetch = [&](int64_t k) {
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int piece = i * kThreads + threadIdx.x;
        held[m][i] = *(const half8*)(from[m] + piece / (kDepth / 8) * stride[m] + k + piece % (kDepth / 8) * 8);
      }
  };
  fetch(0);
  float4v sum[2][2] = {};
  const int wi = wave / 2 * 32, wj = wave % 2 * 32;
  for (int64_t k = 0; k < p.depth; k += kDepth) {
    __syncthreads();
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int piece = i * kThreads + threadIdx.x;
        lds[m][piece_at(piece / (kDepth / 8), piece % (kDepth / 8))] = held[m][i];
      }
    __syncthreads();
    if (k + kDepth < p.depth) fetch(k + kDepth);
#pragma unroll
    for (int q = 0; q < kDepth / 32; ++q) {
      half8 v[4][2];
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int s = 0; s < 2; ++s) v[m][s] = lds[m][piece_at((m < 2 ? wi : wj) + s * 16 + lane % 16, q * 4 + lane / 16)];
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          sum[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[0][a], v[3][b], sum[a][b], 0, 0, 0);
          sum[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[1][a], v[2][b], sum[a][b], 0, 0, 0);
          sum[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[0][a], v[2][b], sum[a][b], 0, 0, 0);
        }
    }
  }
  // A lane has rows 4 (lane / 16) .. + 3 of column lane % 16 of each 16 x 16.
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t i = ti * kTile + wi + a * 16 + lane / 16 * 4 + r, j = tj * kTile + wj + b * 16 + lane % 16;
        float v = sum[a][b][r] * p.factor;
        if constexpr (kMode == kSymmetric) {
          if (p.added.high) {
            const int64_t at = batch * p.added.batch_stride + i * p.added.stride + j;
            v = fmaf(p.added_factor, (float)p.added.high[at] + (float)p.added.low[at], v);
            if (i == j) v += p.diagonal;
          }
          split_store(p.out, batch, i, j, v);
          if (ti != tj) split_store(p.out, batch, j, i, v);
        } else if constexpr (kMode == kBoth) {
          split_store(p.out, batch, i, j, v);
          split_store(p.turned, batch, j, i, v);
        } else {
          if (i < p.rows && j < p.columns)
            ((T*)p.result)[batch * p.result_batch + i * p.row_step + j * p.column_step] = (T)v;
        }
      }
}

// ---- host -------------------------------------------------------------------

int64_t padded(int64_t v) { return (v + kTile - 1) / kTile * kTile; }

// Where the matrices lie in the workspace.
struct Plan {
  int64_t m, n, mp, np;
  size_t partial, x, xt, xt_next, square[5], bytes;
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
  const size_t wide = (size_t)batch * p.mp * p.np * 2 * sizeof(_Float16);
  p.x = take(wide);
  p.xt = take(wide);
  p.xt_next = take(wide);
  for (auto& s : p.square) s = take((size_t)batch * p.mp * p.mp * 2 * sizeof(_Float16));
  p.bytes = at;
  return p;
}

template <typename T>
int orthogonalize(T* out, const T* g, int64_t batch, int64_t rows, int64_t columns, int64_t stride,
                  int64_t batch_stride, int steps, float a, float b, float c, float eps, uint8_t* ws,
                  hipStream_t stream) {
  const Plan pl = plan(batch, rows, columns);
  const bool tall = rows > columns;
  float* partial = (float*)(ws + pl.partial);
  auto matrix = [&](size_t at, int64_t r, int64_t s) {
    _Float16* high = (_Float16*)(ws + at);
    return Split{high, high + batch * r * s, s, r * s};
  };
  const Split x = matrix(pl.x, pl.mp, pl.np);
  Split xt = matrix(pl.xt, pl.np, pl.mp), xt_next = matrix(pl.xt_next, pl.np, pl.mp);
  Split A = matrix(pl.square[0], pl.mp, pl.mp), Z = matrix(pl.square[1], pl.mp, pl.mp),
        U = matrix(pl.square[2], pl.mp, pl.mp), P = matrix(pl.square[3], pl.mp, pl.mp),
        Q = matrix(pl.square[4], pl.mp, pl.mp);
  hipLaunchKernelGGL((k_square_sums<T>), dim3(kNormGroups, (uint32_t)batch), dim3(kThreads), 0, stream, partial, g, rows,
                     columns, stride, batch_stride);
  hipLaunchKernelGGL((k_normalize<T>), dim3((uint32_t)(padded(columns) / kTile), (uint32_t)(padded(rows) / kTile), (uint32_t)batch),
                     dim3(kThreads), 0, stream, tall ? xt : x, tall ? x : xt, g, partial, rows, columns, stride,
                     batch_stride, eps);
  MGB_LAUNCH_CHECK("orthogonalize: scaling");
  const uint32_t mt = (uint32_t)(pl.mp / kTile), nt = (uint32_t)(pl.np / kTile);
  auto square = [&](Split left, Split right, Split to, int64_t depth, float factor, const Split* added = nullptr) {
    Product p = {};
    p.left = left;
    p.right = right;
    p.out = to;
    p.depth = depth;
    p.factor = factor;
    if (added) {
      p.added = *added;
      p.added_factor = b * kScaleZ / kScaleX;
      p.diagonal = a * kScaleZ;
    }
    hipLaunchKernelGGL((k_product<kSymmetric, float>), dim3(mt * (mt + 1) / 2, 1, (uint32_t)batch), dim3(kThreads), 0,
                       stream, p);
  };
  const int segments = (steps + kSegment - 1) / kSegment;
  for (int s = 0; s < segments; ++s) {
    const int length = steps / segments + (s < steps % segments ? 1 : 0);
    square(x, x, A, pl.np, 1.0f / kScaleX);
    for (int k = 0; k < length; ++k) {
      square(A, A, Z, pl.mp, c * kScaleZ / (kScaleX * kScaleX), &A);
      if (k == 0) {
        std::swap(P, Z);
      } else {
        square(Z, P, Q, pl.mp, 1.0f / kScaleZ);
        std::swap(P, Q);
      }
      if (k + 1 < length) {
        const Split z = k == 0 ? P : Z;
        square(z, A, U, pl.mp, 1.0f / kScaleZ);
        square(U, z, A, pl.mp, 1.0f / kScaleZ);
      }
    }
    Product p = {};
    p.left = P;
    p.right = xt;
    p.depth = pl.mp;
    if (s + 1 < segments) {
      // X^T is read whole while the new one is written: two buffers in turn.
      p.out = x;
      p.turned = xt_next;
      p.factor = 1.0f / kScaleZ;
      hipLaunchKernelGGL((k_product<kBoth, float>), dim3(nt, mt, (uint32_t)batch), dim3(kThreads), 0, stream, p);
      std::swap(xt, xt_next);
      continue;
    }
    p.factor = 1.0f / (kScaleZ * kScaleX);
    p.result = out;
    p.rows = pl.m;
    p.columns = pl.n;
    p.row_step = tall ? 1 : columns;
    p.column_step = tall ? columns : 1;
    p.result_batch = rows * columns;
    hipLaunchKernelGGL((k_product<kFinal, T>), dim3(nt, mt, (uint32_t)batch), dim3(kThreads), 0, stream, p);
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
  if (batch == 0 || rows == 0 || columns == 0) return 0;
  MGB_REQUIRE(out && update && workspace, "orthogonalize: null pointer");
  MGB_REQUIRE(workspace_bytes >= mgb_orthogonalize_workspace_bytes(batch, rows, columns),
              "orthogonalize: workspace too small");
  auto run = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
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
