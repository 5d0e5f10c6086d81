// Shared by the encoder's operators (embedding.hip, norm.hip,
// orthogonalize.hip): element types, 16-byte packs at any alignment, sums over
// a group of lanes.  These operators run on the caller's stream and in the
// caller's buffers; they keep nothing between calls.
#pragma once
#include <stdint.h>

#include "device_common.hpp"

namespace mgb {

template <typename T>
struct DTypeOf;
template <>
struct DTypeOf<float> { static constexpr int value = MGB_F32; };
template <>
struct DTypeOf<_Float16> { static constexpr int value = MGB_F16; };
template <>
struct DTypeOf<__bf16> { static constexpr int value = MGB_BF16; };

// 16 bytes of elements.  Rows of any width and stride start anywhere, so packs
// are moved by memcpy: global loads and stores of this chip take any byte
// address, and an aligned pack costs no more for it.
template <typename T>
struct Pack {
  static constexpr int kSize = 16 / sizeof(T);
  T v[kSize];
};

// Elements at .. at + kSize of a row of `dim`, as binary32; beyond the row 0.
// (at may be past the row.)
template <typename T>
__device__ __forceinline__ void load_pack(const T* row, int64_t at, int64_t dim, float* out) {
  constexpr int kSize = Pack<T>::kSize;
  Pack<T> p;
  if (at + kSize <= dim) {
    __builtin_memcpy(&p, row + at, sizeof(p));
#pragma unroll
    for (int e = 0; e < kSize; ++e) out[e] = (float)p.v[e];
  } else if (at < dim) {
#pragma unroll
    for (int e = 0; e < kSize; ++e) out[e] = at + e < dim ? (float)row[at + e] : 0.0f;
  } else {
#pragma unroll
    for (int e = 0; e < kSize; ++e) out[e] = 0.0f;
  }
}

// A parameter row in T or in binary32, whichever `T` the caller passes, taken
// in the pack size of the data.
template <int kSize, typename W>
__device__ __forceinline__ void load_some(const W* row, int64_t at, int64_t dim, float* out) {
  if (at + kSize <= dim) {
    W p[kSize];
    __builtin_memcpy(p, row + at, sizeof(p));
#pragma unroll
    for (int e = 0; e < kSize; ++e) out[e] = (float)p[e];
  } else if (at < dim) {
#pragma unroll
    for (int e = 0; e < kSize; ++e) out[e] = at + e < dim ? (float)row[at + e] : 0.0f;
  } else {
#pragma unroll
    for (int e = 0; e < kSize; ++e) out[e] = 0.0f;
  }
}

// Rounds once, to nearest even.
template <typename T>
__device__ __forceinline__ void store_pack(T* row, int64_t at, int64_t dim, const float* in) {
  constexpr int kSize = Pack<T>::kSize;
  if (at + kSize <= dim) {
    Pack<T> p;
#pragma unroll
    for (int e = 0; e < kSize; ++e) p.v[e] = (T)in[e];
    __builtin_memcpy(row + at, &p, sizeof(p));
  } else if (at < dim) {
#pragma unroll
    for (int e = 0; e < kSize; ++e)
      if (at + e < dim) row[at + e] = (T)in[e];
  }
}

// Sum over aligned groups of kLanes (a power of two, at most a wave); every
// lane of the group gets it.
template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int d = kLanes / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
  return v;
}

// Sum over a workgroup of kThreads; `shared` holds a float per wave.  A second
// call may follow at once: the slots are read before its first barrier ends.
template <int kThreads>
__device__ __forceinline__ float block_sum(float v, float* shared) {
  v = group_sum<kWave>(v);
  __syncthreads();
  if (lane_id() == 0) shared[threadIdx.x / kWave] = v;
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) total += shared[w];
  return total;
}

// Host side: an argument's check that fails leaves its message.
#define MGB_REQUIRE(condition, message)  \
  do {                                   \
    if (!(condition)) {                  \
      ::mgb::set_error(message);         \
      return -1;                         \
    }                                    \
  } while (0)

}  // namespace mgb
