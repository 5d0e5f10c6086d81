// Matrix products by tiles, result = sum over k of left(m, k) right(n, k), for the
// encoder's block (feed_forward.hip) and its 8-bit products (blocks.hip).
//
// A workgroup has a tile of kTileM x kTileN.  A step of the depth is 128 bytes of
// every row (64 16-bit values, 128 8-bit ones); its operands lie in LDS in four
// regions, the upper and lower half of the tile's rows (A0, A1) and of its columns
// (B0, B1), two steps of each.  A wave has a part of all four quarters and works a
// step off in four phases, each one quarter:
//   phase  multiplies   reads into registers      fills (from memory, two steps on)
//     0      A0 B0       B1                        A0
//     1      A0 B1       A1                        B0
//     2      A1 B1       A0 of the next step       B1
//     3      A1 B0       B0 of the next step       A1
// What a phase reads is multiplied in the next; a region is filled again two phases
// after the one that read it, and has five phases to arrive.  (Turned operands, below,
// are read in the phase that multiplies them, each a phase later, and filled again in
// the phase after.)  With eight waves, two a SIMD, the second four are half a phase
// behind: while one wave of a SIMD multiplies, the other reads, and a barrier
// between the halves keeps them so.
//
// An operand's rows either hold the depth without gaps ("straight"), or the depth
// goes from row to row ("turned": the transpose of a matrix as it lies); turned ones
// are transposed by the LDS reads that do so (ds_read_b64_tr_b16).  Chunks of 16
// bytes are permuted within the LDS rows so that lanes that read together hit
// different banks; as loads to LDS go to consecutive places, the lanes fetch their
// chunks permuted.  Whatever lies outside an operand is read as zero by the bounds
// of its buffer descriptor: rows beyond the last, and the depth's end inside a step.
//
// 8,192 x 4,096 x 4,096 in blocks of 8 bits: 126 us, 2.2 PFLOP/s; the gated pair of
// 16,384 x 1,024 to 2 x 4,096 in bfloat16: 318 us, 0.86 PFLOP/s with its epilogue.
#pragma once
#include <type_traits>

#include "encoder_common.hpp"

namespace mgb {
namespace product {

using int4v = __attribute__((ext_vector_type(4))) int;
using int8v = __attribute__((ext_vector_type(8))) int;
using short4v = __attribute__((ext_vector_type(4))) short;
using float4v = __attribute__((ext_vector_type(4))) float;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using SharedBytes = __attribute__((address_space(3))) void*;

struct E4m3 {};  // 8-bit values with a scale (a power of two, its exponent + 127) for each 128

constexpr int kStepBytes = 128;
constexpr int kScaleSteps = 64;  // of 8-bit operands, a workgroup's most

// Binary32 values as three bfloat16 (24 bits) make six products; the three that
// are left out are below 2^-24 of the largest.
__host__ __device__ constexpr int left_part(int pair) { return (0x201100 >> (4 * pair)) & 15; }
__host__ __device__ constexpr int right_part(int pair) { return (0x021010 >> (4 * pair)) & 15; }

// One operand: up to four matrices whose products are added.
struct Operand {
  const char* data[4];
  int64_t stride[4];   // bytes from row to row as they lie
  int64_t part;        // bytes between the parts of binary32 values
  int64_t extent;      // rows (straight), columns (turned) that there are
  int64_t depth;       // values along the depth that there are; straight: whole chunks of 16 bytes
};

constexpr int kMostJobs = 3;
struct Job {
  Operand left, right;
  void* out;
  int64_t out_stride;  // elements
  int64_t rows, columns;
  int64_t partial;     // where its partial sums begin, elements
  uint32_t row_tiles, column_tiles, first_tile;
};

struct Params {
  Job job[kMostJobs];
  int jobs;
  int sources, pairs;
  int64_t depth;             // the larger of the operands'
  uint32_t tiles, splits, first_steps, other_steps;  // the depth's shares: the first, and the others
  float* partials;           // [split][partial_size]
  int64_t partial_size;
  // 8-bit operands: a byte of exponent for each row and step, rows of whole words
  const uint8_t* left_scales;
  const uint8_t* right_scales[2];  // the second for the dual form
  int64_t left_scale_stride, right_scale_stride;
  // the block's epilogues
  float* kept;               // [row][2][hidden], binary32, or null
  char* hidden;              // act(gate) up, in parts
  char* dgate;               // [2][row][stride], in parts: dgate, then dup
  int64_t hidden_stride, hidden_part, gradient_part, gradient_second;  // elements
  int64_t hidden_rest, gradient_rest;  // to what 16-bit values leave, or 0 if that is dropped
  int64_t hidden_columns;    // whole chunks of 8, the rest zeros
  int64_t true_columns;      // columns of `kept`
  int activation;
};

__device__ __forceinline__ void wait_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// vmcnt(n) lgkmcnt(0)
template <int kLoads>
__device__ __forceinline__ void wait_loads() {
  static_assert(kLoads < 64, "vmcnt");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x70 | (kLoads & 15) | (kLoads >> 4) << 14);
  asm volatile("" ::: "memory");
}

template <typename E>
constexpr int element_bytes() { return std::is_same_v<E, E4m3> ? 1 : 2; }

// A 16 x 16 tile's operand of one step: 32 bytes a lane.
struct Fragment {
  int8v v;
  __device__ __forceinline__ int4v half(int h) const {
    return h ? __builtin_shufflevector(v, v, 4, 5, 6, 7) : __builtin_shufflevector(v, v, 0, 1, 2, 3);
  }
};

// sum[4 (lane / 16) + e of right][lane % 16 of left], of half a step
template <typename E>
__device__ __forceinline__ float4v multiply(int4v left, int4v right, float4v sum) {
  if constexpr (std::is_same_v<E, __bf16>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, right), __builtin_bit_cast(bf16x8, left), sum,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, right), __builtin_bit_cast(f16x8, left), sum, 0,
                                                  0, 0);
}

// The scales' lowest bytes count.
__device__ __forceinline__ float4v multiply8(const Fragment& left, const Fragment& right, int left_scale, int right_scale,
                                             float4v sum) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(right.v, left.v, sum, 0, 0, 0, right_scale, 0, left_scale);
}

// A tile's shape: waves kWavesM x kWavesN; of each region's rows a wave has kRowsM or kRowsN.
template <int kM, int kN, int kWM, int kWN>
struct Tile {
  static constexpr int kTileM = kM, kTileN = kN, kWavesM = kWM, kWavesN = kWN;
  static constexpr int kWaves = kWM * kWN, kThreads = kWaves * kWave;
  static constexpr int kHalfM = kM / 2, kHalfN = kN / 2;
  static constexpr int kRowsM = kHalfM / kWM, kRowsN = kHalfN / kWN;
  static constexpr int kTilesM = kRowsM / 16, kTilesN = kRowsN / 16;
  static constexpr int kRegionM = kHalfM * kStepBytes, kRegionN = kHalfN * kStepBytes;
  static constexpr int kLoadsM = kRegionM / (kThreads * 16), kLoadsN = kRegionN / (kThreads * 16);
  static constexpr int kBytes = 4 * kRegionM + 4 * kRegionN;
  static constexpr bool kAlternate = kWaves == 8;
  static_assert(kLoadsM * kThreads * 16 == kRegionM && kLoadsN * kThreads * 16 == kRegionN, "whole loads");
};
using Large = Tile<256, 256, 2, 4>;
using Medium = Tile<128, 128, 2, 2>;
using Small = Tile<64, 64, 2, 2>;

// The tile of a workgroup: an eighth of the workgroups (a chiplet's, which takes
// every eighth) has a stretch of an order that goes by bands of kBand tile rows,
// column by column, so that what a chiplet works on at one time shares operands.
// The shares of the depth follow each other, the longest first.
constexpr uint32_t kBand = 4;
__device__ __forceinline__ bool find_tile(const Params& p, uint32_t* job, uint32_t* ti, uint32_t* tj, uint32_t* split) {
  const uint32_t each = (p.tiles + 7) / 8, local = blockIdx.x / 8;
  uint32_t tile = blockIdx.x % 8 * each + local % each, j = 0;
  *split = local / each;
  if (tile >= p.tiles || *split >= p.splits) return false;
  while (j + 1 < (uint32_t)p.jobs && tile >= p.job[j + 1].first_tile) ++j;
  tile -= p.job[j].first_tile;
  const uint32_t rows = p.job[j].row_tiles, columns = p.job[j].column_tiles;
  const uint32_t band = tile / (kBand * columns), in = tile % (kBand * columns);
  const uint32_t height = rows - band * kBand < kBand ? rows - band * kBand : kBand;
  *job = j;
  *ti = band * kBand + in % height;
  *tj = in / height;
  return true;
}

// Straight columns in pairs of 16 x 16 tiles: column 8 a + 4 j + b of 32 is row 4 a + b of
// tile j, so that a lane's sums of a pair are 8 columns that follow each other.
template <bool kTurned, typename S>
constexpr bool paired() { return !kTurned && S::kTilesN % 2 == 0; }
// The chunks of a row are permuted by this, which differs among the 8 rows that lanes
// read together: 8 that follow each other, or 8 a + b for a pair's.
template <bool kPairs>
__device__ __forceinline__ int straight_key(int row) {
  return kPairs ? (row & 3) | (row >> 3 & 1) << 2 : row & 7;
}

// How the 32-byte granules of a turned row in LDS are permuted: the 32 lanes that
// are served together read four rows from 4 k on and the four 8 rows further, 32 bytes
// of each, which are to lie in different banks (of 256 bytes) whatever the rows' length.
template <int kGranules>
__device__ __forceinline__ int turned_key(int row) {
  if constexpr (kGranules == 8) return (row & 3) | (row >> 3 & 1) << 2;
  if constexpr (kGranules == 4) return (row >> 1 & 1) | (row >> 3 & 1) << 1;
  return row >> 3 & 1;
}

// 16 columns and the step's depth of turned rows in LDS, transposed, for tiles at `at`
// (bytes of LDS): four reads of 8 values of the depth each, 4 x 16 values at a time.  The
// compiler would wait for all loads to LDS before its own form of these reads; here
// the wait for the reads alone stands in the same statement.
template <int kPitch, int kOffset, int kTiles>
__device__ __forceinline__ void read_turned(const uint32_t* at, Fragment* f) {
  using int2v = __attribute__((ext_vector_type(2))) int;
  // Offsets of the depth's 4 rows from 0, 4, 32 and 36 on.
  constexpr int k0 = kOffset, k1 = kOffset + 4 * kPitch, k2 = kOffset + 32 * kPitch, k3 = kOffset + 36 * kPitch;
  static_assert(k3 < 65536, "the instruction's offsets");
  int2v v[kTiles][4];
#define MGB_READS(t)                                      \
  "ds_read_b64_tr_b16 %[a" #t "], %[at" #t "] offset:%[k0]\n" \
  "ds_read_b64_tr_b16 %[b" #t "], %[at" #t "] offset:%[k1]\n" \
  "ds_read_b64_tr_b16 %[c" #t "], %[at" #t "] offset:%[k2]\n" \
  "ds_read_b64_tr_b16 %[d" #t "], %[at" #t "] offset:%[k3]\n"
#define MGB_OUT(t) [a##t] "=&v"(v[t][0]), [b##t] "=&v"(v[t][1]), [c##t] "=&v"(v[t][2]), [d##t] "=&v"(v[t][3])
#define MGB_OFFSETS [k0] "n"(k0), [k1] "n"(k1), [k2] "n"(k2), [k3] "n"(k3)
  if constexpr (kTiles == 4) {
    asm volatile(MGB_READS(0) MGB_READS(1) MGB_READS(2) MGB_READS(3) "s_waitcnt lgkmcnt(0)"
                 : MGB_OUT(0), MGB_OUT(1), MGB_OUT(2), MGB_OUT(3)
                 : [at0] "v"(at[0]), [at1] "v"(at[1]), [at2] "v"(at[2]), [at3] "v"(at[3]), MGB_OFFSETS
                 : "memory");
  } else if constexpr (kTiles == 2) {
    asm volatile(MGB_READS(0) MGB_READS(1) "s_waitcnt lgkmcnt(0)"
                 : MGB_OUT(0), MGB_OUT(1)
                 : [at0] "v"(at[0]), [at1] "v"(at[1]), MGB_OFFSETS
                 : "memory");
  } else {
    static_assert(kTiles == 1, "tiles of a wave");
    asm volatile(MGB_READS(0) "s_waitcnt lgkmcnt(0)" : MGB_OUT(0) : [at0] "v"(at[0]), MGB_OFFSETS : "memory");
  }
#undef MGB_READS
#undef MGB_OUT
#undef MGB_OFFSETS
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int k = 0; k < 8; ++k) f[t].v[k] = v[t][k / 2][k % 2];
}

// What is read of an operand: a cursor that goes over its steps, the products of
// the parts, and the matrices.  All of it is the same for a workgroup's lanes.
template <bool kTurned, bool kPairs, int kHalf, int kLoads, int kWaves>
struct Reader {
  const char* from[2];       // the regions' first rows, now
  int64_t left[2];           // bytes from there to the end of what the region has
  int64_t stride, depth;
  uint32_t offset[kLoads];   // this lane's, from `from`
  uint32_t chunk;            // straight: where in the step the lane's 16 bytes are

  __device__ __forceinline__ void lanes(int64_t row_stride) {
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      if constexpr (!kTurned) {
        const int row = (q * kWaves + wave) * 8 + lane / 8;
        chunk = ((lane % 8) ^ straight_key<kPairs>(row)) * 16;  // (the same for all q)
        offset[q] = (uint32_t)(row * row_stride) + chunk;
      } else {
        // A row of kHalf values is kHalf / 8 chunks.
        constexpr int kChunks = kHalf / 8;
        const int slot = (q * kWaves + wave) * kWave + lane, row = slot / kChunks, at = slot % kChunks;
        offset[q] = (uint32_t)(row * row_stride) + ((at ^ (2 * turned_key<kChunks / 2>(row))) * 16);
      }
    }
  }
};

// The exponents of the 8-bit operands' rows, of up to 64 steps: words of a step's
// left rows, then of its right rows.
template <typename S>
struct Scales {
  static constexpr int kWordsM = 2 * S::kTilesM / 4 > 0 ? 2 * S::kTilesM / 4 : 1;  // of a lane's rows
  static constexpr int kWordsN = 2 * S::kTilesN / 4 > 0 ? 2 * S::kTilesN / 4 : 1;
  static constexpr int kM = S::kWavesM * 16 * kWordsM, kN = S::kWavesN * 16 * kWordsN;
  static constexpr int kBytes = (kM + kN) * 4;  // a step's

  template <int kHalf, int kRows, int kTiles, int kWords, bool kPairs>
  static __host__ __device__ __forceinline__ int place(int row) {  // byte
    const int half = row / kHalf, wave = row % kHalf / kRows, in = row % kRows;
    const int tile = kPairs ? in / 32 * 2 + in / 4 % 2 : in / 16;
    const int lane = kPairs ? in % 32 / 8 * 4 + in % 4 : in % 16;
    const int byte = half * kTiles + tile;
    return ((wave * 16 + lane) * kWords + byte / 4) * 4 + byte % 4;
  }
  // The step whose exponents are read while one of `steps` is multiplied: a panel ends at its
  // last.
  static __host__ __device__ __forceinline__ uint32_t ahead(uint32_t step, uint32_t steps) {
    return step + 1 < steps ? step + 1 : step;
  }
  // Words of a row that hold steps begin to end, and one of them, `at` of all the tile's rows'.
  static __host__ __device__ __forceinline__ int words(uint32_t begin, uint32_t end) {
    return (int)((end + 3) / 4 - begin / 4);
  }
  static __host__ __device__ __forceinline__ void fill_word(char* panel, int at, const Params& p, int64_t row0, int64_t rows,
                                                            int64_t column0, int64_t columns, bool dual, uint32_t begin,
                                                            uint32_t end) {
    const int each = words(begin, end), row = at / each, quad = at % each;
    const uint8_t* from = nullptr;
    int to;
    if (row < S::kTileM) {
      if (row0 + row < rows) from = p.left_scales + (row0 + row) * p.left_scale_stride;
      to = place<S::kHalfM, S::kRowsM, S::kTilesM, kWordsM, false>(row);
    } else {
      const int r = row - S::kTileM;
      const int64_t column = column0 + (dual ? r % S::kHalfN : r);
      if (column < columns) from = p.right_scales[dual ? r / S::kHalfN : 0] + column * p.right_scale_stride;
      to = kM * 4 + place<S::kHalfN, S::kRowsN, S::kTilesN, kWordsN, paired<false, S>()>(r);
    }
    // (Rows are whole words, and shares begin anywhere: the first and the last may have other
    // shares' steps.)
    const uint32_t first = (begin / 4 + quad) * 4, word = from ? *(const uint32_t*)(from + first) : 0x7f7f7f7fu;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
      if (first + e >= begin && first + e < end) panel[(first + e - begin) * kBytes + to] = (char)(word >> (8 * e));
  }
  static __device__ __forceinline__ void fill(char* panel, const Params& p, int64_t row0, int64_t rows, int64_t column0,
                                              int64_t columns, bool dual, uint32_t begin, uint32_t end) {
    for (int at = threadIdx.x; at < (S::kTileM + S::kTileN) * words(begin, end); at += S::kThreads)
      fill_word(panel, at, p, row0, rows, column0, columns, dual, begin, end);
  }
};

template <typename E, bool kLeftTurned, bool kRightTurned, typename S, class Finish>
__global__ __launch_bounds__(S::kThreads, 2) void k_product(Params p) {
  constexpr bool k8 = std::is_same_v<E, E4m3>;
  constexpr int kBytes = element_bytes<E>();
  constexpr int kStep = kStepBytes / kBytes;  // elements
  static_assert(!k8 || (!kLeftTurned && !kRightTurned), "8-bit operands lie straight");
  // Straight operands are read a phase before they are multiplied (A0 and A1 in
  // registers of their own); the turned ones' addresses leave no registers for that.
  constexpr bool kAhead = !kLeftTurned && !kRightTurned;
  constexpr bool kPairs = paired<kRightTurned, S>();
  __shared__ __attribute__((aligned(1024))) char lds[S::kBytes + (k8 ? Scales<S>::kBytes * kScaleSteps : 0)];

  uint32_t which, ti, tj, split;
  if (!find_tile(p, &which, &ti, &tj, &split)) return;
  const Job& job = p.job[which];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / S::kWavesN, wn = wave % S::kWavesN;

  // ---- memory to LDS
  Reader<kLeftTurned, false, S::kHalfM, S::kLoadsM, S::kWaves> left;
  Reader<kRightTurned, kPairs, S::kHalfN, S::kLoadsN, S::kWaves> right;
  const int64_t row0 = (int64_t)ti * S::kTileM;
  // The dual form has the columns of one matrix in B0 and the same ones of the other in B1.
  const int64_t column0 = (int64_t)tj * (Finish::kDual ? S::kHalfN : S::kTileN);
  left.depth = job.left.depth;
  right.depth = job.right.depth;
  const uint32_t each = p.depth > 0 ? (uint32_t)((p.depth + kStep - 1) / kStep) : 1;
  const uint32_t all = each * p.pairs * p.sources;
  const uint32_t begin = split ? p.first_steps + (split - 1) * p.other_steps : 0, share = split ? p.other_steps : p.first_steps;
  const uint32_t end = begin + share < all ? begin + share : all;

  // The cursor: step k of the depth, of a product of parts, of a matrix.
  uint32_t ahead = begin;  // the next step to fetch
  uint32_t k = begin % each, pair = begin / each % p.pairs, source = begin / each / p.pairs;
  auto place = [&] {
    const int s = Finish::kDual ? 0 : source;
    auto base = [&](const Operand& o, int matrix, int part) { return o.data[matrix] + part * o.part; };
    left.stride = job.left.stride[s];
    right.stride = job.right.stride[s];
    const int lp = p.pairs > 1 ? left_part(pair) : 0, rp = p.pairs > 1 ? right_part(pair) : 0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t row = row0 + r * S::kHalfM;
      if constexpr (!kLeftTurned) {
        left.from[r] = base(job.left, s, lp) + row * left.stride + (int64_t)k * kStepBytes;
        const int64_t rows = job.left.extent - row < S::kHalfM ? job.left.extent - row : S::kHalfM;
        left.left[r] = rows > 0 ? (rows - 1) * left.stride + (left.depth * kBytes - (int64_t)k * kStepBytes) : 0;
      } else {
        left.from[r] = base(job.left, s, lp) + (int64_t)k * kStep * left.stride + row * kBytes;
        left.left[r] = row < job.left.extent ? (job.left.extent - row) * kBytes : 0;
      }
      const int64_t column = column0 + (Finish::kDual ? 0 : r * S::kHalfN);
      const int matrix = Finish::kDual ? r : s;
      const int64_t stride = job.right.stride[matrix];
      if constexpr (!kRightTurned) {
        right.from[r] = base(job.right, matrix, rp) + column * stride + (int64_t)k * kStepBytes;
        const int64_t rows = job.right.extent - column < S::kHalfN ? job.right.extent - column : S::kHalfN;
        right.left[r] = rows > 0 ? (rows - 1) * stride + (right.depth * kBytes - (int64_t)k * kStepBytes) : 0;
      } else {
        right.from[r] = base(job.right, matrix, rp) + (int64_t)k * kStep * stride + column * kBytes;
        right.left[r] = column < job.right.extent ? (job.right.extent - column) * kBytes : 0;
      }
    }
  };
  if (begin < end) place();
  // (Both matrices of an operand lie at the same distance: the entries see to that.)
  left.lanes(job.left.stride[0]);
  right.lanes(job.right.stride[0]);
  auto advance = [&] {
    ++ahead;
    if (++k < each) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        left.from[r] += kLeftTurned ? kStep * left.stride : kStepBytes;
        right.from[r] += kRightTurned ? kStep * right.stride : kStepBytes;
        if (!kLeftTurned && left.left[r] > 0) left.left[r] -= kStepBytes;
        if (!kRightTurned && right.left[r] > 0) right.left[r] -= kStepBytes;
      }
    } else {
      k = 0;
      if (++pair == (uint32_t)p.pairs) {
        pair = 0;
        ++source;
      }
      if (ahead < end) place();
    }
  };
  // Loads of steps beyond the last have an empty buffer: they read nothing and fill
  // with zeros, and the count of loads in flight stays what the waits take it for.
  auto fetch = [&](auto& reader, int r, char* to, auto turned, auto loads) {
    int64_t bytes = reader.left[r];
    if constexpr (decltype(turned)::value) {
      const int64_t depth = reader.depth - (int64_t)k * kStep < kStep ? reader.depth - (int64_t)k * kStep : kStep;
      bytes = bytes > 0 && depth > 0 ? bytes + (depth - 1) * reader.stride : 0;
    }
    if (ahead >= end) bytes = 0;
    const __amdgpu_buffer_rsrc_t buffer =
        __builtin_amdgcn_make_buffer_rsrc((void*)reader.from[r], 0, (int)bytes, 0x00020000);
#pragma unroll
    for (int q = 0; q < decltype(loads)::value; ++q) {
      uint32_t offset = reader.offset[q];
      if constexpr (!decltype(turned)::value)
        offset = (int64_t)k * kStepBytes + reader.chunk < reader.depth * kBytes ? offset : 0x80000000u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (SharedBytes)(to + (q * S::kWaves + wave) * (kWave * 16)), 16,
                                               (int)offset, 0, 0, 0);
    }
  };
  using LeftTurned = std::bool_constant<kLeftTurned>;
  using RightTurned = std::bool_constant<kRightTurned>;
  using LoadsM = std::integral_constant<int, S::kLoadsM>;
  using LoadsN = std::integral_constant<int, S::kLoadsN>;
  char* const lds_right = lds + 4 * S::kRegionM;
  auto left_region = [&](int r, int stage) { return lds + (r * 2 + stage) * S::kRegionM; };
  auto right_region = [&](int r, int stage) { return lds_right + (r * 2 + stage) * S::kRegionN; };
  auto fetch_left = [&](int r, int stage) { fetch(left, r, left_region(r, stage), LeftTurned{}, LoadsM{}); };
  auto fetch_right = [&](int r, int stage) { fetch(right, r, right_region(r, stage), RightTurned{}, LoadsN{}); };

  // ---- LDS to registers
  // Straight: lane l has row l % 16 (of a pair 8 (l % 16 / 4) + l % 4), chunks l / 16 and
  // l / 16 + 4 of it.  Turned: its 8 values of a half are 8 l / 16 .. + 7 of the depth, by
  // two reads of 4 x 16 that transpose: lane l gives the place of row l % 16 / 4, columns
  // l % 4 * 4 .. + 3.
  auto straight = [&](const char* region, int first_row, int t, auto pairs) {
    int4v part[2];
    constexpr bool kIn = decltype(pairs)::value;
    const int row = kIn ? lane % 16 / 4 * 8 + lane % 4 : lane % 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int chunk = (lane / 16 ^ (lane & 7)) ^ (h * 4);
      part[h] = *(const int4v*)(region + (first_row + row) * kStepBytes + chunk * 16 +
                                (kIn ? t / 2 * 32 + t % 2 * 4 : t * 16) * kStepBytes);
    }
    Fragment f;
    f.v = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return f;
  };
  auto turned_places = [&](uint32_t* at, const char* first_region, int first_row, int tiles, auto half_rows) {
    constexpr int kPitch = decltype(half_rows)::value * 2, kGranules = decltype(half_rows)::value / 16;
    const int row = lane / 16 * 8 + lane % 16 / 4;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)first_region;
#pragma unroll
    for (int t = 0; t < tiles; ++t)
      at[t] = base + row * kPitch + ((first_row / 16 + t) ^ turned_key<kGranules>(row)) * 32 + lane % 4 * 8;
  };
  uint32_t left_at[S::kTilesM], right_at[S::kTilesN];
  if constexpr (kLeftTurned) turned_places(left_at, lds, wm * S::kRowsM, S::kTilesM, std::integral_constant<int, S::kHalfM>{});
  if constexpr (kRightTurned) turned_places(right_at, lds_right, wn * S::kRowsN, S::kTilesN, std::integral_constant<int, S::kHalfN>{});
  Fragment a[kAhead ? 2 : 1][S::kTilesM], b[2][S::kTilesN];
  auto take_left = [&](auto r, auto stage) {
    constexpr int kR = decltype(r)::value, kStage = decltype(stage)::value;
    if constexpr (kLeftTurned) {
      read_turned<S::kHalfM * 2, (kR * 2 + kStage) * S::kRegionM, S::kTilesM>(left_at, a[0]);
    } else {
#pragma unroll
      for (int i = 0; i < S::kTilesM; ++i)
        a[kAhead ? kR : 0][i] = straight(left_region(kR, kStage), wm * S::kRowsM, i, std::false_type{});
    }
  };
  auto take_right = [&](Fragment* to, auto r, auto stage) {
    constexpr int kR = decltype(r)::value, kStage = decltype(stage)::value;
    if constexpr (kRightTurned) {
      read_turned<S::kHalfN * 2, (kR * 2 + kStage) * S::kRegionN, S::kTilesN>(right_at, to);
    } else {
#pragma unroll
      for (int j = 0; j < S::kTilesN; ++j)
        to[j] = straight(right_region(kR, kStage), wn * S::kRowsN, j, std::bool_constant<kPairs>{});
    }
  };

  // A row's exponents of a step: bytes kTilesM x + i of words that lanes l % 16 of the
  // rows' waves read, for all of its steps.
  using Panel = Scales<S>;
  struct Words {
    uint32_t left[Panel::kWordsM], right[Panel::kWordsN];
  };
  Words scales = {}, next_scales = {};
  auto read_scales = [&](uint32_t step) {
    Words w = {};
    if constexpr (k8) {
      const uint32_t* words = (const uint32_t*)(lds + S::kBytes) + step * (Panel::kBytes / 4);
      __builtin_memcpy(w.left, words + (wm * 16 + lane % 16) * Panel::kWordsM, sizeof(w.left));
      __builtin_memcpy(w.right, words + Panel::kM + (wn * 16 + lane % 16) * Panel::kWordsN, sizeof(w.right));
    }
    return w;
  };

  float4v sum[2][2][S::kTilesM][S::kTilesN] = {};
  // Tiles i and j of a quarter; without a 8-bit step, half of it.
  auto multiply_tile = [&](int x, int y, int i, int j, int h, const Fragment& right) {
    if constexpr (k8) {
      const int l = x * S::kTilesM + i, r = y * S::kTilesN + j;
      if (h == 0)
        sum[x][y][i][j] = multiply8(a[kAhead ? x : 0][i], right, (int)(scales.left[l / 4] >> (l % 4 * 8)),
                                    (int)(scales.right[r / 4] >> (r % 4 * 8)), sum[x][y][i][j]);
    } else {
      sum[x][y][i][j] = multiply<E>(a[kAhead ? x : 0][i].half(h), right.half(h), sum[x][y][i][j]);
    }
  };

  // ---- the steps
  constexpr int kFlight = (kAhead ? 5 : 6) * S::kLoadsM;  // loads issued after the region that is waited for
  static_assert(S::kLoadsM == S::kLoadsN, "regions of one size");
  auto order = [] { __builtin_amdgcn_sched_barrier(0); };
  // Matrix instructions have no order of their own among barriers and loads: empty
  // statements that name the sums hold them within a phase.
  auto hold = [&](int x, int y) {
#pragma unroll
    for (int i = 0; i < S::kTilesM; ++i)
#pragma unroll
      for (int j = 0; j < S::kTilesN; ++j) asm volatile("" : "+v"(sum[x][y][i][j]));
  };
  // The regions that the next phase reads are there, and what this one read is out of LDS.
  auto arrived = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xf70 | (kFlight & 15) | (kFlight >> 4) << 14);  // vmcnt(kFlight)
    asm volatile("" ::: "memory");
  };
  auto taken = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
  };
  // The end of a phase, after its reads and loads are issued.
  auto multiply_quarter = [&](int x, int y, const Fragment* right) {
    order();
    if constexpr (!kAhead) taken();
    if constexpr (!kAhead || S::kAlternate) {
      arrived();
      wait_barrier();
    }
    if constexpr (S::kAlternate) __builtin_amdgcn_s_setprio(1);
    order();
    hold(x, y);
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // (those of one sum far apart: one waits for the other)
#pragma unroll
      for (int i = 0; i < S::kTilesM; ++i)
#pragma unroll
        for (int j = 0; j < S::kTilesN; ++j) multiply_tile(x, y, i, j, h, right[j]);
      order();
    }
    hold(x, y);
    order();
    if constexpr (S::kAlternate) __builtin_amdgcn_s_setprio(0);
    if constexpr (kAhead) taken();
    if constexpr (kAhead && !S::kAlternate) arrived();
    if constexpr (kAhead || S::kAlternate) wait_barrier();
    order();
  };
  using Zero = std::integral_constant<int, 0>;
  using One = std::integral_constant<int, 1>;
  const uint32_t steps = end > begin ? end - begin : 0;
  auto step = [&](auto stage_constant, uint32_t t) {
    constexpr int kStage = decltype(stage_constant)::value;
    using Now = std::integral_constant<int, kStage>;
    using Next = std::integral_constant<int, 1 - kStage>;
    Fragment *const now = b[kStage], *const other = b[1 - kStage];
    if constexpr (kAhead) {
      take_right(other, One{}, Now{});
      fetch_left(0, kStage);
      multiply_quarter(0, 0, now);
      take_left(One{}, Now{});
      fetch_right(0, kStage);
      multiply_quarter(0, 1, other);
      take_left(Zero{}, Next{});
      fetch_right(1, kStage);
      multiply_quarter(1, 1, other);
      take_right(other, Zero{}, Next{});
      next_scales = read_scales(Panel::ahead(t, steps));
      fetch_left(1, kStage);
      advance();
      multiply_quarter(1, 0, now);
      scales = next_scales;
    } else {
      fetch_right(0, kStage);
      take_left(Zero{}, Now{});
      multiply_quarter(0, 0, now);
      fetch_left(0, kStage);
      take_right(other, One{}, Now{});
      multiply_quarter(0, 1, other);
      fetch_right(1, kStage);
      take_left(One{}, Now{});
      multiply_quarter(1, 1, other);
      fetch_left(1, kStage);
      advance();
      take_right(other, Zero{}, Next{});
      multiply_quarter(1, 0, now);
    }
  };
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if constexpr (kAhead) fetch_left(0, s);
    fetch_right(0, s);
    if constexpr (!kAhead) fetch_left(0, s);
    fetch_right(1, s);
    fetch_left(1, s);
    advance();
  }
  if constexpr (k8) {
    Panel::fill(lds + S::kBytes, p, row0, job.left.extent, column0, job.right.extent, Finish::kDual, begin, end);
    wait_loads<0>();
  } else {
    wait_loads<kFlight>();
  }
  wait_barrier();
  scales = read_scales(0);
  take_right(b[0], Zero{}, Zero{});
  if constexpr (kAhead) take_left(Zero{}, Zero{});
  wait_loads<kFlight>();
  wait_barrier();
  if constexpr (S::kAlternate)
    if (wave >= S::kWaves / 2) wait_barrier();
  for (uint32_t t = 0; t + 2 <= steps; t += 2) {
    step(std::integral_constant<int, 0>{}, t);
    step(std::integral_constant<int, 1>{}, t + 1);
  }
  if (steps % 2) step(std::integral_constant<int, 0>{}, steps - 1);
  if constexpr (S::kAlternate)
    if (wave < S::kWaves / 2) wait_barrier();
  // Nothing may land in LDS after the workgroup has ended.
  wait_loads<0>();

  // ---- what becomes of the sums: a lane has 4 or, of pairs, 8 columns of a row
  const Finish finish(p, job, split);
  constexpr int kCount = kPairs ? 8 : 4, kGroups = S::kTilesN * 4 / kCount, kHalves = Finish::kDual ? 1 : 2;
  constexpr int kItems = 2 * S::kTilesM * kGroups * kHalves, kDeep = Finish::kDeep < kItems ? Finish::kDeep : kItems;
  const int64_t m0 = row0 + wm * S::kRowsM + lane % 16, n0 = column0 + wn * S::kRowsN + lane / 16 * kCount;
  auto row_of = [&](int item) {
    return m0 + item / (S::kTilesM * kGroups * kHalves) * S::kHalfM + item / (kGroups * kHalves) % S::kTilesM * 16;
  };
  auto column_of = [&](int item) { return n0 + item / kHalves % kGroups * (4 * kCount) + item % kHalves * S::kHalfN; };
  if constexpr (Finish::kBlocks) {
    // Results in 8 bits: a tile's 128 columns are a block.  Each wave's largest values
    // of its rows meet in LDS.
    static_assert(Finish::kDual && kPairs && S::kHalfN == 128, "a block a tile");
    float* const tops = (float*)lds;
    wait_barrier();
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < S::kTilesM; ++i) {
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < S::kTilesN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = finish.value(sum[x][0][i][j][e], sum[x][1][i][j][e]);
            sum[x][0][i][j][e] = v;
            top = fmaxf(top, fabsf(v) < INFINITY ? fabsf(v) : 0.0f);
          }
        top = fmaxf(top, __shfl_xor(top, 16, kWave));
        top = fmaxf(top, __shfl_xor(top, 32, kWave));
        if (lane < 16) tops[wn * S::kTileM + x * S::kHalfM + wm * S::kRowsM + i * 16 + lane] = top;
      }
    wait_loads<0>();
    wait_barrier();
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int i = 0; i < S::kTilesM; ++i) {
        const int row = x * S::kHalfM + wm * S::kRowsM + i * 16 + lane % 16;
        if (row0 + row >= job.rows) continue;
        float top = 0.0f, v[S::kTilesN * 4];
#pragma unroll
        for (int w = 0; w < S::kWavesN; ++w) top = fmaxf(top, tops[w * S::kTileM + row]);
#pragma unroll
        for (int e = 0; e < S::kTilesN * 4; ++e) v[e] = sum[x][0][i][e / 4][e % 4];
        finish.store(row0 + row, n0, tj, v, top, wn == 0 && lane < 16);
      }
  } else {
    auto finish_tile = [&](auto whole) {
      // What the end reads of memory is on its way kDeep items ahead.
      typename Finish::template Loaded<kCount> ring[kDeep];
#pragma unroll
      for (int item = 0; item < kDeep; ++item)
        finish.template load<kCount, decltype(whole)::value>(ring[item], row_of(item), column_of(item));
#pragma unroll
      for (int item = 0; item < kItems; ++item) {
        const int x = item / (S::kTilesM * kGroups * kHalves), i = item / (kGroups * kHalves) % S::kTilesM;
        const int j = item / kHalves % kGroups * (kCount / 4), y = item % kHalves;
        float v[2][kCount];
#pragma unroll
        for (int e = 0; e < kCount; ++e) {
          v[0][e] = sum[x][y][i][j + e / 4][e % 4];
          if constexpr (Finish::kDual) v[1][e] = sum[x][1][i][j + e / 4][e % 4];
        }
        finish.template store<kCount, decltype(whole)::value>(row_of(item), column_of(item), v[0], v[1], ring[item % kDeep]);
        if (item + kDeep < kItems)
          finish.template load<kCount, decltype(whole)::value>(ring[item % kDeep], row_of(item + kDeep), column_of(item + kDeep));
      }
    };
    if (row0 + S::kTileM <= job.rows && column0 + (Finish::kDual ? S::kHalfN : S::kTileN) <= job.columns)
      finish_tile(std::true_type{});
    else
      finish_tile(std::false_type{});
  }
}

// Values of a row, to the type rounded once; without kWhole those beyond `columns` are
// not stored.
template <int kCount, bool kWhole, typename T>
__device__ __forceinline__ void store_some(T* row, int64_t n, int64_t columns, const float* v) {
  T r[kCount];
#pragma unroll
  for (int e = 0; e < kCount; ++e) r[e] = (T)v[e];
  if (kWhole || n + kCount <= columns) {
    __builtin_memcpy(row + n, r, sizeof(r));
  } else {
#pragma unroll
    for (int e = 0; e < kCount; ++e)
      if (n + e < columns) row[n + e] = r[e];
  }
}

// What ends a tile: store() takes the sums (of a dual form both matrices') of kCount
// columns of a row from n on, and what load() fetched before.  kWhole: the tile lies
// within the result.
struct Plainly {
  static constexpr bool kDual = false, kBlocks = false;
  static constexpr int kDeep = 1;
  template <int kCount>
  struct Loaded {};
  template <int kCount, bool kWhole, typename L>
  __device__ __forceinline__ void load(L&, int64_t, int64_t) const {}
};

template <typename T>
struct Store : Plainly {
  T* out;
  int64_t stride, rows, columns;
  __device__ __forceinline__ Store(const Params&, const Job& job, uint32_t)
      : out((T*)job.out), stride(job.out_stride), rows(job.rows), columns(job.columns) {}
  template <int kCount, bool kWhole, typename L>
  __device__ __forceinline__ void store(int64_t m, int64_t n, const float* v, const float*, const L&) const {
    if (kWhole || m < rows) store_some<kCount, kWhole>(out + m * stride, n, columns, v);
  }
};

// A share of the depth, added up by k_join.
struct Partial : Plainly {
  float* out;
  int64_t rows, columns;
  __device__ __forceinline__ Partial(const Params& p, const Job& job, uint32_t split)
      : out(p.partials + split * p.partial_size + job.partial), rows(job.rows), columns(job.columns) {}
  template <int kCount, bool kWhole, typename L>
  __device__ __forceinline__ void store(int64_t m, int64_t n, const float* v, const float*, const L&) const {
    if (kWhole || m < rows) store_some<kCount, kWhole>(out + m * columns, n, columns, v);
  }
};

}  // namespace product
}  // namespace mgb
