// Shared by the encoder's operators (embedding.hip, norm.hip,
// orthogonalize.hip): element types, 16-byte packs at any alignment, sums over
// a group of lanes.  These operators run on the caller's stream and in the
// caller's buffers; they keep nothing between calls.
#pragma once
#include <stdint.h>

#include <type_traits>

#include "device_common.hpp"

namespace mgb {

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

// kSize elements as they lie in memory, 16 bytes or one element: loaded without
// a branch, so that many are in flight, and converted afterwards.
template <typename T, int kSize>
struct Raw {
  static_assert(kSize == 1 || kSize == Pack<T>::kSize, "a pack or an element");
  using Bits = std::conditional_t<kSize == 1, std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>,
                                  __attribute__((ext_vector_type(4))) uint32_t>;
  Bits bits;
  __device__ __forceinline__ void load(const T* from) { __builtin_memcpy(&bits, from, sizeof(bits)); }
  __device__ __forceinline__ void keep_if(bool keep) {
    if constexpr (kSize == 1) {
      bits = keep ? bits : Bits(0);
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) bits[w] = keep ? bits[w] : 0u;
    }
  }
  __device__ __forceinline__ void get(float* out) const {
    T v[kSize];
    __builtin_memcpy(v, &bits, sizeof(bits));
#pragma unroll
    for (int e = 0; e < kSize; ++e) out[e] = (float)v[e];
  }
  __device__ __forceinline__ void put(const float* in, T* to) {  // rounds to nearest even
    T v[kSize];
#pragma unroll
    for (int e = 0; e < kSize; ++e) v[e] = (T)in[e];
    __builtin_memcpy(to, v, sizeof(v));
  }
};

// sum += v, and sum += a + b.  The chip adds binary16 to binary32 in one
// instruction if it is a multiply-add (`one` is 1, from where the compiler does
// not see it), and two bfloat16 by a dot product with (1, 1): 16 instructions
// for two packs of eight, where conversions and additions take 32.
template <typename T, int kSize>
__device__ __forceinline__ void add_one(const Raw<T, kSize>& v, float one, float* sum) {
  T x[kSize];
  __builtin_memcpy(x, &v.bits, sizeof(v.bits));
#pragma unroll
  for (int e = 0; e < kSize; ++e)
    if constexpr (std::is_same_v<T, _Float16>) sum[e] = fmaf((float)x[e], one, sum[e]);
    else sum[e] += (float)x[e];
}

template <typename T, int kSize>
__device__ __forceinline__ void add_two(const Raw<T, kSize>& a, const Raw<T, kSize>& b, float one, float* sum) {
  if constexpr (std::is_same_v<T, __bf16> && kSize > 1) {
    using Pair = __attribute__((ext_vector_type(2))) __bf16;
    const uint32_t ones_bits = 0x3f803f80;
    Pair ones;
    __builtin_memcpy(&ones, &ones_bits, 4);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t low = __builtin_amdgcn_perm(b.bits[w], a.bits[w], 0x05040100u);
      const uint32_t high = __builtin_amdgcn_perm(b.bits[w], a.bits[w], 0x07060302u);
      Pair l, h;
      __builtin_memcpy(&l, &low, 4);
      __builtin_memcpy(&h, &high, 4);
      sum[2 * w] = __builtin_amdgcn_fdot2_f32_bf16(l, ones, sum[2 * w], false);
      sum[2 * w + 1] = __builtin_amdgcn_fdot2_f32_bf16(h, ones, sum[2 * w + 1], false);
    }
  } else {
    add_one<T, kSize>(a, one, sum);
    add_one<T, kSize>(b, one, sum);
  }
}

// 1, as a value of the run.
__device__ __forceinline__ float runtime_one() {
  float one = 1.0f;
  asm volatile("" : "+v"(one));
  return one;
}

// Sum over aligned groups of kLanes (a power of two, at most a wave); every
// lane of the group gets it.  Within 16 lanes the exchanges are lane moves, which
// take no turn of LDS's: lanes 1 and 2 apart by quad permutations, and, as the
// lanes of a quad then hold one value, and those of two quads, 4 and 8 apart by
// mirrored halves of a row and mirrored rows.
template <int kCtrl>
__device__ __forceinline__ float lane_move(float v) {
  return __uint_as_float(dpp_move<kCtrl, 0xf>(__float_as_uint(v)));
}

template <int kLanes>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr (kLanes >= 64) v += __shfl_xor(v, 32, kWave);
  if constexpr (kLanes >= 32) v += __shfl_xor(v, 16, kWave);
  if constexpr (kLanes >= 2) v += lane_move<0xb1>(v);
  if constexpr (kLanes >= 4) v += lane_move<0x4e>(v);
  if constexpr (kLanes >= 8) v += lane_move<0x141>(v);
  if constexpr (kLanes >= 16) v += lane_move<0x140>(v);
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

// Two sums at once; `shared` holds two floats per wave.
template <int kThreads>
__device__ __forceinline__ void block_sums(float& a, float& b, float* shared) {
  constexpr int kWaves = kThreads / kWave;
  a = group_sum<kWave>(a);
  b = group_sum<kWave>(b);
  __syncthreads();
  if (lane_id() == 0) {
    shared[threadIdx.x / kWave] = a;
    shared[kWaves + threadIdx.x / kWave] = b;
  }
  __syncthreads();
  // (A lane a wave's: 2 kWaves registers at once would cost a second workgroup.)
  a = group_sum<kWaves>(shared[lane_id() % kWaves]);
  b = group_sum<kWaves>(shared[kWaves + lane_id() % kWaves]);
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
