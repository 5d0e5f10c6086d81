// Products of binary32 values, each three bfloat16 (product.hpp), where tiles are small.
// k_product goes over its operands once for each of the six products of parts; here a
// step is 32 of the depth with all parts of both operands, so that memory, LDS and
// registers see each part once where that way sees it twice.  Three steps lie in LDS:
// one is multiplied, the next is on its way or there, and the third is filled once all
// waves have left it, which one barrier a step sees to.
//
// The gradients of 2,003 x 200 x 777: 74 us (83, as the parts came, and 104 with k_product's
// tiles of these sizes); those of 2,048 x 1,024 x 4,096 641 us, 161 TFLOP/s (a library's
// binary32 product 152).
// What bounds small ones are the loads to LDS, 64 bytes of a row each, at 21 bytes a
// cycle and compute unit.
#pragma once
#include "product.hpp"

namespace mgb {
namespace product {

// Waves kWavesM x kWavesN; each has kRowsM of the left rows and kRowsN of the right
// rows of both halves (of a dual form the two matrices).
template <int kM, int kN, int kWM, int kWN>
struct PartTile {
  static constexpr int kTileM = kM, kTileN = kN, kHalfN = kN / 2, kWavesN = kWN;
  static constexpr int kWaves = kWM * kWN, kThreads = kWaves * kWave;
  static constexpr int kRowsM = kM / kWM, kRowsN = kHalfN / kWN;
  static constexpr int kTilesM = kRowsM / 16, kTilesN = kRowsN / 16;
  static constexpr int kParts = 3, kDepth = 32, kStages = 3;
  static constexpr int kPartM = kM * kDepth * 2, kPartN = kN * kDepth * 2;  // bytes
  static constexpr int kStage = kParts * (kPartM + kPartN);
  static_assert(kPartM == kThreads * 16 && kPartN == kThreads * 16, "a load a part");
};
using PartMedium = PartTile<128, 128, 2, 4>;
using PartSmall = PartTile<64, 64, 2, 2>;

// Tiles of 16 columns and the step's depth of turned rows, transposed: two reads each.
// (The wait stands in the statement, as in read_turned.)
template <int kPitch, int kOffset, int kTiles>
__device__ __forceinline__ void read_turned_step(const uint32_t* at, int4v* f) {
  using int2v = __attribute__((ext_vector_type(2))) int;
  constexpr int k0 = kOffset, k1 = kOffset + 4 * kPitch;
  static_assert(k1 < 65536, "the instruction's offsets");
  int2v v[kTiles][2];
#define MGB_READS(t)                                          \
  "ds_read_b64_tr_b16 %[a" #t "], %[at" #t "] offset:%[k0]\n" \
  "ds_read_b64_tr_b16 %[b" #t "], %[at" #t "] offset:%[k1]\n"
#define MGB_OUT(t) [a##t] "=&v"(v[t][0]), [b##t] "=&v"(v[t][1])
#define MGB_OFFSETS [k0] "n"(k0), [k1] "n"(k1)
  if constexpr (kTiles == 4) {
    asm volatile(MGB_READS(0) MGB_READS(1) MGB_READS(2) MGB_READS(3) "s_waitcnt lgkmcnt(0)"
                 : MGB_OUT(0), MGB_OUT(1), MGB_OUT(2), MGB_OUT(3)
                 : [at0] "v"(at[0]), [at1] "v"(at[1]), [at2] "v"(at[2]), [at3] "v"(at[3]), MGB_OFFSETS
                 : "memory");
  } else {
    static_assert(kTiles == 2, "tiles of a wave");
    asm volatile(MGB_READS(0) MGB_READS(1) "s_waitcnt lgkmcnt(0)"
                 : MGB_OUT(0), MGB_OUT(1)
                 : [at0] "v"(at[0]), [at1] "v"(at[1]), MGB_OFFSETS
                 : "memory");
  }
#undef MGB_READS
#undef MGB_OUT
#undef MGB_OFFSETS
#pragma unroll
  for (int t = 0; t < kTiles; ++t) f[t] = __builtin_shufflevector(v[t][0], v[t][1], 0, 1, 2, 3);
}

template <bool kLeftTurned, bool kRightTurned, typename S, class Finish>
__global__ __launch_bounds__(S::kThreads, 2) void k_parts(Params p) {
  constexpr bool kDual = Finish::kDual;
  static_assert(!kDual || !kRightTurned, "the dual form's matrices lie straight");
  __shared__ __attribute__((aligned(1024))) char lds[S::kStages * S::kStage];
  uint32_t which, ti, tj, split;
  if (!find_tile(p, &which, &ti, &tj, &split)) return;
  const Job& job = p.job[which];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / S::kWavesN, wn = wave % S::kWavesN;
  const int64_t row0 = (int64_t)ti * S::kTileM, column0 = (int64_t)tj * (kDual ? S::kHalfN : S::kTileN);

  // ---- memory to LDS: a wave fills 1 KB of each part, 16 straight rows or a stretch
  // of the turned ones.
  const uint32_t each = p.depth > 0 ? (uint32_t)((p.depth + S::kDepth - 1) / S::kDepth) : 1, all = each * p.sources;
  const uint32_t begin = split ? p.first_steps + (split - 1) * p.other_steps : 0, share = split ? p.other_steps : p.first_steps;
  const uint32_t end = begin + share < all ? begin + share : all;
  uint32_t ahead = begin, k = begin % each, source = begin / each;

  const int straight_row = lane / 4, straight_chunk = lane % 4 ^ (straight_row >> 1 & 3);
  auto turned_offset = [&](auto side, int64_t stride) {
    constexpr int kChunks = decltype(side)::value / 8;
    const int slot = wave * kWave + lane, row = slot / kChunks, at = slot % kChunks;
    return (uint32_t)(row * stride) + (at ^ (2 * turned_key<kChunks / 2>(row))) * 16;
  };
  // (Both matrices of an operand lie at the same distance: the entries see to that.)
  uint32_t left_offset, right_offset;
  if constexpr (kLeftTurned) left_offset = turned_offset(std::integral_constant<int, S::kTileM>{}, job.left.stride[0]);
  else left_offset = (uint32_t)(straight_row * job.left.stride[0]) + straight_chunk * 16;
  if constexpr (kRightTurned) right_offset = turned_offset(std::integral_constant<int, S::kTileN>{}, job.right.stride[0]);
  else right_offset = (uint32_t)(straight_row * job.right.stride[0]) + straight_chunk * 16;

  auto fetch_side = [&](const Operand& o, int matrix, int64_t first, auto turned, uint32_t offset, char* to, int part_bytes) {
    const int64_t stride = o.stride[matrix];
    const char* from = o.data[matrix];
    int64_t bytes;
    if constexpr (decltype(turned)::value) {
      const int64_t depth = o.depth - (int64_t)k * S::kDepth < S::kDepth ? o.depth - (int64_t)k * S::kDepth : S::kDepth;
      from += (int64_t)k * S::kDepth * stride + first * 2;
      bytes = first < o.extent && depth > 0 ? (o.extent - first) * 2 + (depth - 1) * stride : 0;
    } else {
      const int64_t rows = o.extent - first < 16 ? o.extent - first : 16;
      from += first * stride + (int64_t)k * (S::kDepth * 2);
      bytes = rows > 0 ? (rows - 1) * stride + (o.depth * 2 - (int64_t)k * (S::kDepth * 2)) : 0;
      if ((int64_t)k * (S::kDepth * 2) + straight_chunk * 16 >= o.depth * 2) offset = 0x80000000u;
    }
    if (ahead >= end || bytes < 0) bytes = 0;
#pragma unroll
    for (int part = 0; part < S::kParts; ++part) {
      const __amdgpu_buffer_rsrc_t buffer = __builtin_amdgcn_make_buffer_rsrc((void*)(from + part * o.part), 0, (int)bytes, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (SharedBytes)(to + part * part_bytes + wave * (kWave * 16)), 16, (int)offset,
                                               0, 0, 0);
    }
  };
  // Steps beyond the last read nothing and fill with zeros: the count of loads in
  // flight stays what the waits take it for.
  auto fetch = [&](int stage) {
    char* const to = lds + stage * S::kStage;
    const int s = source < (uint32_t)p.sources ? source : 0;
    fetch_side(job.left, kDual ? 0 : s, row0 + (kLeftTurned ? 0 : wave * 16), std::bool_constant<kLeftTurned>{}, left_offset, to,
               S::kPartM);
    const int matrix = kDual ? wave / (S::kWaves / 2) : s, rows = kDual ? wave % (S::kWaves / 2) : wave;
    fetch_side(job.right, matrix, column0 + (kRightTurned ? 0 : rows * 16), std::bool_constant<kRightTurned>{}, right_offset,
               to + S::kParts * S::kPartM, S::kPartN);
    ++ahead;
    if (++k == each) {
      k = 0;
      ++source;
    }
  };

  // ---- LDS to registers
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  auto turned_place = [&](int first_row, int t, auto side) {
    constexpr int kPitch = decltype(side)::value * 2, kGranules = decltype(side)::value / 16;
    const int row = lane / 16 * 8 + lane % 16 / 4;
    return lds_at + row * kPitch + ((first_row / 16 + t) ^ turned_key<kGranules>(row)) * 32 + lane % 4 * 8;
  };
  const int straight_at = lane % 16 * 64 + (lane / 16 ^ (lane % 16 >> 1 & 3)) * 16;
  int4v a[S::kParts][S::kTilesM], b[S::kParts][2 * S::kTilesN];
  auto take = [&](int stage) {
    const char* const left = lds + stage * S::kStage;
    const char* const right = left + S::kParts * S::kPartM;
    if constexpr (kLeftTurned) {
      uint32_t at[S::kTilesM];
#pragma unroll
      for (int i = 0; i < S::kTilesM; ++i)
        at[i] = turned_place(wm * S::kRowsM, i, std::integral_constant<int, S::kTileM>{}) + stage * S::kStage;
      read_turned_step<S::kTileM * 2, 0, S::kTilesM>(at, a[0]);
      read_turned_step<S::kTileM * 2, S::kPartM, S::kTilesM>(at, a[1]);
      read_turned_step<S::kTileM * 2, 2 * S::kPartM, S::kTilesM>(at, a[2]);
    } else {
#pragma unroll
      for (int part = 0; part < S::kParts; ++part)
#pragma unroll
        for (int i = 0; i < S::kTilesM; ++i)
          a[part][i] = *(const int4v*)(left + part * S::kPartM + (wm * S::kRowsM + i * 16) * 64 + straight_at);
    }
    if constexpr (kRightTurned) {
      constexpr int kFirst = S::kParts * S::kPartM;
      uint32_t at[2 * S::kTilesN];
#pragma unroll
      for (int j = 0; j < 2 * S::kTilesN; ++j)
        at[j] = turned_place(j / S::kTilesN * S::kHalfN + wn * S::kRowsN, j % S::kTilesN, std::integral_constant<int, S::kTileN>{}) +
                stage * S::kStage + kFirst;
      read_turned_step<S::kTileN * 2, 0, 2 * S::kTilesN>(at, b[0]);
      read_turned_step<S::kTileN * 2, S::kPartN, 2 * S::kTilesN>(at, b[1]);
      read_turned_step<S::kTileN * 2, 2 * S::kPartN, 2 * S::kTilesN>(at, b[2]);
    } else {
#pragma unroll
      for (int part = 0; part < S::kParts; ++part)
#pragma unroll
        for (int j = 0; j < 2 * S::kTilesN; ++j)
          b[part][j] = *(const int4v*)(right + part * S::kPartN +
                                       (j / S::kTilesN * S::kHalfN + wn * S::kRowsN + j % S::kTilesN * 16) * 64 + straight_at);
    }
  };

  // ---- the steps
  float4v sum[S::kTilesM][2 * S::kTilesN] = {};
  fetch(0);
  fetch(1);
  int stage = 0;
  for (uint32_t t = begin; t < end; ++t) {
    // This step's loads are there, and every wave has the last step's out of LDS.
    wait_loads<2 * S::kParts>();
    wait_barrier();
    fetch(stage == 0 ? 2 : stage - 1);
    take(stage);
    stage = stage == 2 ? 0 : stage + 1;
#pragma unroll
    for (int pair = 0; pair < 6; ++pair)
#pragma unroll
      for (int i = 0; i < S::kTilesM; ++i)
#pragma unroll
        for (int j = 0; j < 2 * S::kTilesN; ++j)
          sum[i][j] = multiply<__bf16>(a[left_part(pair)][i], b[right_part(pair)][j], sum[i][j]);
  }
  // Nothing may land in LDS after the workgroup has ended.
  wait_loads<0>();

  // ---- what becomes of the sums: they meet in LDS, from where a lane has 8 columns of a
  // row and 8 lanes or more have what lies together.
  constexpr int kPitch = S::kTileN + 4;
  static_assert(S::kTileM * kPitch * 4 <= S::kStages * S::kStage, "the sums fit");
  float* const sums = (float*)lds;
  wait_barrier();
#pragma unroll
  for (int i = 0; i < S::kTilesM; ++i)
#pragma unroll
    for (int j = 0; j < 2 * S::kTilesN; ++j)
      *(float4v*)(sums + (wm * S::kRowsM + i * 16 + lane % 16) * kPitch + j / S::kTilesN * S::kHalfN + wn * S::kRowsN +
                  j % S::kTilesN * 16 + lane / 16 * 4) = sum[i][j];
  wait_loads<0>();
  wait_barrier();
  const Finish finish(p, job, split);
  constexpr int kColumns = kDual ? S::kHalfN : S::kTileN, kLanes = kColumns / 8, kRows = S::kThreads / kLanes;
  constexpr int kItems = S::kTileM / kRows, kDeep = Finish::kDeep < kItems ? Finish::kDeep : kItems;
  const int row = threadIdx.x / kLanes, column = threadIdx.x % kLanes * 8;
  auto finish_tile = [&](auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    typename Finish::template Loaded<8> ring[kDeep];
#pragma unroll
    for (int item = 0; item < kDeep; ++item)
      finish.template load<8, kWhole>(ring[item], row0 + row + item * kRows, column0 + column);
#pragma unroll
    for (int item = 0; item < kItems; ++item) {
      const float* const from = sums + (row + item * kRows) * kPitch + column;
      float v[2][8];
      __builtin_memcpy(v[0], __builtin_assume_aligned(from, 16), sizeof(v[0]));
      if constexpr (kDual) __builtin_memcpy(v[1], __builtin_assume_aligned(from + S::kHalfN, 16), sizeof(v[1]));
      finish.template store<8, kWhole>(row0 + row + item * kRows, column0 + column, v[0], v[1], ring[item % kDeep]);
      if (item + kDeep < kItems)
        finish.template load<8, kWhole>(ring[item % kDeep], row0 + row + (item + kDeep) * kRows, column0 + column);
    }
  };
  if (row0 + S::kTileM <= job.rows && column0 + kColumns <= job.columns) finish_tile(std::true_type{});
  else finish_tile(std::false_type{});
}

}  // namespace product
}  // namespace mgb
