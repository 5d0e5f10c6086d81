// Embedding lookup with scaling, one token a row or a row's tokens summed, and
// its gradient by sorted tokens.
//
//   y[r] = s sum_j W[t_rj]          (a token outside the table adds nothing)
//   dW[v] = s sum_{(r, j): t_rj = v} dy[r]
//
// The lookup reads each named row of W once from memory and again from cache;
// its gradient is the same sum turned round.  Sorted by token (stably, so a
// table row's terms keep the order of the tokens), that sum is a walk over
// segments: every group of lanes takes the same number of sorted tokens, so a
// frequent token costs no more than rare ones, and what a segment leaves in
// several groups is joined in order.  No sum depends on the order of atomics.
//
// Measured (us, one MI355X, whose copies reach 5.1 TB/s): lookup 262,144 x 100
// bfloat16 tokens of a table of 25,600 x 64 153, 8,191 rows of 1,024 6.2 (at the
// copies' rate); gradient of 65,536 x 100 tokens 181 (sorts 88, sums 79, join 15,
// windows 7), of 16,411 tokens and rows of 1,024 52, of 256 x 100 tokens 13.
#include <type_traits>

#include "encoder_common.hpp"

namespace mgb {
namespace {

constexpr int kThreads = 256;

// ---- lookup ---------------------------------------------------------------

// Tokens a lane has in flight at once, and the lanes that fetch their numbers.
constexpr int kAhead = 8;

// Columns: a lane holds kSize of a row's, a pack or, in rows narrower than a
// pack, one.  The last pack of a row that is no whole number of packs begins
// early, so that it ends with the row: two lanes then compute the same columns
// and store the same values.
template <int kLanes, int kSize>
__device__ __forceinline__ bool columns_of(int lane, int64_t dim, int64_t* at) {
  const int64_t nominal = ((int64_t)blockIdx.y * kLanes + lane) * kSize;
  *at = nominal < dim - kSize ? nominal : dim - kSize;
  return nominal < dim;
}

// A lane's share of kAhead numbers that its kLanes neighbours walk together (one
// of them, where there are kAhead lanes or more), and all of them from the shares.
template <int kLanes>
constexpr int kShare = kLanes >= kAhead ? 1 : kAhead;

template <int kLanes, typename I>
__device__ __forceinline__ I share_of(const I* mine, int j) {
  if constexpr (kLanes >= kAhead) return __shfl(mine[0], j, kAhead);
  else return mine[j];
}

// kLanes lanes share a row (further columns are other workgroups', blockIdx.y);
// `split` groups share a row's tokens, kAhead in turn, and are joined through
// LDS in their order.  O: byte offsets into the table, 32 bits where it is less
// than 4 GB (20,000 x 100 tokens of 64 columns 21.1 us, with 64 bits 25.9).  Many tokens are bound by what the chiplets' caches give the compute
// units: 262,144 x 100 rows of 128 bytes take 153 us, 22 TB/s (90 % of the lines
// hit there).  Instructions per token come next, so the lane that fetches a token
// also checks it and finds its row.  Gathers from slices of the table in LDS, with
// the sums of 1,024 rows in registers, took 156 us: they save 60 % of the lines, but
// add barriers, and the additions alone are 85 us of vector instructions.
template <typename T, typename I, typename O, int kLanes, int kSize>
__global__ __launch_bounds__(kThreads) void k_lookup_pooled(T* __restrict__ out, const T* __restrict__ weight,
                                                            const I* __restrict__ tokens, int64_t rows, int64_t bag,
                                                            uint32_t vocabulary, int64_t dim, int64_t stride_bytes,
                                                            float scale, int split) {
  __shared__ float shared[kThreads * kSize];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int part = group % split, rows_here = kThreads / kLanes / split;
  constexpr int kMine = kShare<kLanes>;
  const float one = runtime_one();
  int64_t at;
  const bool active = columns_of<kLanes, kSize>(lane, dim, &at);
  const O column = (O)(at * (int64_t)sizeof(T));
  const char* table = (const char*)weight;
  for (int64_t base = (int64_t)blockIdx.x * rows_here; base < rows; base += (int64_t)gridDim.x * rows_here) {
    const int64_t row = base + group / split;
    float sum[kSize] = {};
    if (row < rows) {
      const I* ids = tokens + row * bag;
      for (int64_t first = (int64_t)part * kAhead; first < bag; first += (int64_t)split * kAhead) {
        O offset[kMine];
        bool present[kMine], all = true;
#pragma unroll
        for (int j = 0; j < kMine; ++j) {
          const int64_t t = first + (kMine == 1 ? lane % kAhead : j);
          const int64_t id = t < bag ? (int64_t)ids[t] : -1;
          present[j] = (uint64_t)id < vocabulary;
          offset[j] = present[j] ? (O)(id * stride_bytes) : O(0);
          all = all && present[j];
        }
        // (Lanes beyond the columns hold shares too: no exchange is theirs to miss.)
        O from[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) from[j] = share_of<kLanes>(offset, j) + column;
        const bool whole = __all(all);
        bool keep[kAhead];
        if (!whole) {
          uint32_t mine[kMine];
#pragma unroll
          for (int j = 0; j < kMine; ++j) mine[j] = present[j];
#pragma unroll
          for (int j = 0; j < kAhead; ++j) keep[j] = share_of<kLanes>(mine, j) != 0;
        }
        if (active) {
          Raw<T, kSize> v[kAhead];
#pragma unroll
          for (int j = 0; j < kAhead; ++j) v[j].load((const T*)(table + from[j]));
          if (!whole) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) v[j].keep_if(keep[j]);
          }
#pragma unroll
          for (int j = 0; j < kAhead; j += 2) add_two<T, kSize>(v[j], v[j + 1], one, sum);
        }
      }
    }
    if (split > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < kSize; ++e) shared[threadIdx.x * kSize + e] = sum[e];
      __syncthreads();
      if (part == 0)
        for (int p = 1; p < split; ++p)
#pragma unroll
          for (int e = 0; e < kSize; ++e) sum[e] += shared[(threadIdx.x + p * kLanes) * kSize + e];
    }
    if (part == 0 && row < rows && active) {
#pragma unroll
      for (int e = 0; e < kSize; ++e) sum[e] *= scale;
      Raw<T, kSize>().put(sum, out + row * dim + at);
    }
  }
}

// One token a row, or none.
template <typename T, typename I, int kLanes, int kSize>
__global__ __launch_bounds__(kThreads) void k_lookup(T* __restrict__ out, const T* __restrict__ weight,
                                                     const I* __restrict__ tokens, int64_t rows, int64_t bag,
                                                     int64_t vocabulary, int64_t dim, int64_t stride, float scale) {
  constexpr int kGroups = kThreads / kLanes;
  int64_t at;
  if (!columns_of<kLanes, kSize>(threadIdx.x % kLanes, dim, &at)) return;
  for (int64_t row = (int64_t)blockIdx.x * kGroups + threadIdx.x / kLanes; row < rows;
       row += (int64_t)gridDim.x * kGroups) {
    const int64_t id = bag ? (int64_t)tokens[row] : -1;
    const bool present = id >= 0 && id < vocabulary;
    Raw<T, kSize> v;
    float x[kSize];
    v.load(weight + at + (present ? id : 0) * stride);
    v.keep_if(present);
    v.get(x);
#pragma unroll
    for (int e = 0; e < kSize; ++e) x[e] *= scale;
    v.put(x, out + row * dim + at);
  }
}

// ---- gradient: stable sort of the tokens -----------------------------------
//
// A token becomes one entry, its table row above, its row of `grad` below, in
// 32 bits where both fit (else 64), and the entries are sorted by table row.
// Tokens that name no row carry the number `vocabulary` and sort last.
//
// Where a table row has many tokens and `grad` is larger than a chiplet's
// cache, the rows of `grad` are cut into windows that are sorted and summed
// apart, window w by the workgroups of chiplet w mod 8: its cache then holds
// what its tokens gather.
//
// 6.55 million tokens in two passes: counts 11 and 9 us, scatters 34 and 29 (the
// ranking by ballots, not the 52 MB moved, which are 10 us), scans 3 to 5.

constexpr int kDigitBits = 8, kDigits = 1 << kDigitBits;
constexpr int kChiplets = 8;

struct Sort {
  uint32_t vocabulary, bag;
  uint32_t rows, window;  // rows of grad, and of a window
  uint32_t windows, tiles;  // tiles of a window
  int row_bits, digit_bits;
  uint64_t tokens;        // of a whole window: window * bag
};

// A window's number of tokens; the last windows may hold fewer, or none.
__device__ __forceinline__ uint32_t window_tokens(const Sort& s, uint32_t window) {
  const uint64_t begin = (uint64_t)window * s.window;
  if (begin >= s.rows) return 0;
  const uint32_t rows = s.rows - (uint32_t)begin;
  return (rows < s.window ? rows : s.window) * s.bag;
}

// Workgroups of one chiplet follow each other at distance kChiplets; the windows
// are a multiple of it or divide it.
__device__ __forceinline__ void window_of(uint32_t windows, uint32_t parts, uint32_t block, uint32_t* window,
                                          uint32_t* part) {
  const uint32_t side_by_side = windows < kChiplets ? windows : kChiplets, turn = block / side_by_side;
  *window = turn / parts * side_by_side + block % side_by_side;
  *part = turn % parts;
}

template <typename E, typename I>
struct TokenEntries {
  const I* tokens;
  __device__ E operator()(const Sort& s, uint32_t window, uint32_t i) const {
    const int64_t id = (int64_t)tokens[(uint64_t)window * s.tokens + i];
    const uint32_t key = id >= 0 && id < (int64_t)s.vocabulary ? (uint32_t)id : s.vocabulary;
    return (E)key << s.row_bits | i / s.bag;
  }
};
template <typename E>
struct SortedEntries {
  const E* entries;
  __device__ E operator()(const Sort& s, uint32_t window, uint32_t i) const {
    return entries[(uint64_t)window * s.tokens + i];
  }
};

template <typename E>
__device__ __forceinline__ uint32_t digit_of(const Sort& s, E entry, int pass) {
  return (uint32_t)(entry >> (s.row_bits + pass * s.digit_bits)) & ((1u << s.digit_bits) - 1);
}

// The lanes among `of` whose digit is this lane's, by ballots.
__device__ __forceinline__ uint64_t equal_digits(uint32_t digit, uint64_t of) {
  uint64_t same = of;
#pragma unroll
  for (int b = 0; b < kDigitBits; ++b) {
    const uint32_t bit = 0u - (digit >> b & 1);  // all ones, or none
    const uint64_t ones = __ballot(bit != 0), all = (uint64_t)bit << 32 | bit;
    same &= ~(ones ^ all);
  }
  return same;
}

// Ranks `kRounds` entries of each lane (a wave's entries follow each other, 64
// a round) among the workgroup's entries of equal digit, in their order:
// in a round, lanes of equal digits find each other by ballots; counts[wave][]
// holds what the wave has had.  Leaves in `counts` each wave's offset within
// the digit and in totals[] the digits' numbers.  rank is within the wave.
template <int kWaves, int kRounds, typename E>
__device__ __forceinline__ void rank_digits(const Sort& s, int pass, const E* entry, uint32_t first, uint32_t count,
                                            uint32_t (*counts)[kDigits], uint32_t* totals, uint32_t* rank) {
  const uint32_t lane = lane_id(), wave = threadIdx.x / kWave;
  for (uint32_t d = threadIdx.x; d < kWaves * kDigits; d += kWaves * kWave) (&counts[0][0])[d] = 0;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const uint32_t digit = digit_of(s, entry[k], pass);
    const bool valid = first + k * kWave < count;
    const uint64_t valids = __ballot(valid);
    if (valids == 0) break;  // the whole wave
    const uint64_t same = equal_digits(digit, valids);
    const int leader = same ? __ffsll((unsigned long long)same) - 1 : (int)lane;
    uint32_t before = 0;
    if (valid && leader == (int)lane) before = atomicAdd(&counts[wave][digit], (uint32_t)__popcll(same));
    before = __shfl(before, leader, kWave);
    rank[k] = before + (uint32_t)__popcll(same & ((1ull << lane) - 1));
  }
  __syncthreads();
  for (uint32_t d = threadIdx.x; d < kDigits; d += kWaves * kWave) {
    uint32_t offset = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t c = counts[w][d];
      counts[w][d] = offset;
      offset += c;
    }
    totals[d] = offset;
  }
  __syncthreads();
}

// totals[] to its exclusive prefix sums, by the first kDigits lanes; the others
// take part in the barriers.
__device__ __forceinline__ void scan_digits(uint32_t* totals, uint32_t* shared) {
  const uint32_t v = threadIdx.x < kDigits ? totals[threadIdx.x] : 0;
  uint32_t all;
  const uint32_t before = block_exclusive_u32(v, shared, &all);
  if (threadIdx.x < kDigits) totals[threadIdx.x] = before;
  __syncthreads();
}

// Bytes that workgroups beyond a sort's own set to zero while the sort, which
// leaves memory idle, runs: what later launches count in, and the table.
struct Clear {
  uint8_t* at[2];
  uint64_t bytes[2];
};

template <int kBlock>
__device__ __forceinline__ void clear(const Clear& c, uint32_t block, uint32_t blocks) {
  const uint4 zero = {};
  for (int k = 0; k < 2; ++k) {
    const uint64_t step = (uint64_t)blocks * kBlock * sizeof(zero);
    for (uint64_t i = ((uint64_t)block * kBlock + threadIdx.x) * sizeof(zero); i < c.bytes[k]; i += step) {
      if (i + sizeof(zero) <= c.bytes[k]) {
        __builtin_memcpy(c.at[k] + i, &zero, sizeof(zero));
      } else {
        for (uint64_t b = i; b < c.bytes[k]; ++b) c.at[k][b] = 0;
      }
    }
  }
}

constexpr int kSortThreads = 512, kSortWaves = kSortThreads / kWave;
constexpr uint32_t kFewTiles = 64;  // at most, for the sort without scans between its passes

// counts[window][digit][tile], or with kFew (one window) counts[tile][digit];
// workgroups beyond the tiles clear.
template <typename F, int kRounds, bool kFew>
__global__ __launch_bounds__(kSortThreads) void k_sort_count(uint32_t* __restrict__ counts, F from, Sort s, int pass,
                                                             Clear zero) {
  const uint32_t blocks = s.windows * s.tiles;
  if (blockIdx.x >= blocks) {
    clear<kSortThreads>(zero, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  __shared__ uint32_t count[kDigits];
  if (threadIdx.x < kDigits) count[threadIdx.x] = 0;
  __syncthreads();
  uint32_t window, tile;
  window_of(s.windows, s.tiles, blockIdx.x, &window, &tile);
  const uint32_t n = window_tokens(s, window), first = tile * (kRounds * kSortThreads) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < kRounds; ++k)
    if (first + k * kSortThreads < n) atomicAdd(&count[digit_of(s, from(s, window, first + k * kSortThreads), pass)], 1u);
  __syncthreads();
  if (threadIdx.x < kDigits)
    counts[kFew ? (uint64_t)tile * kDigits + threadIdx.x
                : ((uint64_t)window * kDigits + threadIdx.x) * s.tiles + tile] = count[threadIdx.x];
}

// One digit's counts become the offsets of its tiles within the digit.
__global__ __launch_bounds__(kThreads) void k_sort_scan(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals,
                                                        uint32_t tiles) {
  __shared__ uint32_t shared[kThreads / kWave + 1];
  uint32_t* mine = counts + (uint64_t)blockIdx.x * tiles;
  uint32_t before = 0;
  for (uint32_t base = 0; base < tiles; base += kThreads) {
    const uint32_t t = base + threadIdx.x;
    const uint32_t v = t < tiles ? mine[t] : 0;
    uint32_t total;
    const uint32_t offset = block_exclusive_u32(v, shared, &total);
    if (t < tiles) mine[t] = before + offset;
    before += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = before;
}

// A tile's entries are brought in order in LDS, so that those of one digit
// leave it as one run.  With few tiles (kFew) a workgroup adds up the tiles'
// counts itself, and counts the next pass's digits where its entries go: three
// launches for two passes instead of six (whole gradients, us: 25,600 tokens 24.5 and
// 32.0, 131,000 tokens 39.8 and 39.0).
template <typename E, typename F, int kRounds, bool kFew>
__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(E* __restrict__ out, F from,
                                                               const uint32_t* __restrict__ counts,
                                                               const uint32_t* __restrict__ totals,
                                                               uint32_t* __restrict__ next_counts, Sort s, int pass,
                                                               Clear zero) {
  constexpr uint32_t kTile = kRounds * kSortThreads;
  const uint32_t blocks = s.windows * s.tiles;
  if (blockIdx.x >= blocks) {
    clear<kSortThreads>(zero, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  __shared__ uint32_t count[kSortWaves][kDigits];
  __shared__ uint32_t here[kDigits], to[kDigits], before[kDigits];
  __shared__ uint32_t shared[kSortWaves + 1];
  __shared__ E entries[kTile];
  uint32_t window, tile;
  window_of(s.windows, s.tiles, blockIdx.x, &window, &tile);
  const uint32_t all = window_tokens(s, window), begin = tile * kTile;
  if (begin >= all) return;  // the last window's tiles may be fewer
  const uint32_t n = all - begin < kTile ? all - begin : kTile;
  const uint32_t first = threadIdx.x / kWave * (kRounds * kWave) + lane_id();
  E entry[kRounds];
  uint32_t rank[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) entry[k] = first + k * kWave < n ? from(s, window, begin + first + k * kWave) : 0;
  if constexpr (kFew) {
    // Two lanes a digit, tiles in turn, all loads in flight.
    const uint32_t d = threadIdx.x % kDigits, half = threadIdx.x / kDigits;
    uint32_t sum = 0, ahead = 0;
#pragma unroll
    for (uint32_t k = 0; k < kFewTiles / 2; ++k) {
      const uint32_t t = half + 2 * k, c = t < s.tiles ? counts[t * kDigits + d] : 0;
      sum += c;
      ahead += t < tile ? c : 0;
    }
    if (half == 0) {
      to[d] = sum;
      before[d] = ahead;
    }
    __syncthreads();
    if (half == 1) {
      to[d] += sum;
      before[d] += ahead;
    }
  } else if (threadIdx.x < kDigits) {
    to[threadIdx.x] = totals[window * kDigits + threadIdx.x];
    before[threadIdx.x] = counts[((uint64_t)window * kDigits + threadIdx.x) * s.tiles + tile];
  }
  rank_digits<kSortWaves, kRounds>(s, pass, entry, first, n, count, here, rank);
  scan_digits(here, shared);
  scan_digits(to, shared);
  if (threadIdx.x < kDigits) to[threadIdx.x] += before[threadIdx.x] - here[threadIdx.x];
#pragma unroll
  for (int k = 0; k < kRounds; ++k)
    if (first + k * kWave < n) {
      const uint32_t d = digit_of(s, entry[k], pass);
      entries[here[d] + count[threadIdx.x / kWave][d] + rank[k]] = entry[k];
    }
  __syncthreads();
  E* mine = out + (uint64_t)window * s.tokens;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const uint32_t i = k * kSortThreads + threadIdx.x;
    if (i < n) {
      const E e = entries[i];
      const uint32_t place = to[digit_of(s, e, pass)] + i;
      mine[place] = e;
      if (kFew && next_counts) atomicAdd(&next_counts[place / kTile * kDigits + digit_of(s, e, pass + 1)], 1u);
    }
  }
}

__global__ __launch_bounds__(kThreads) void k_clear(Clear zero) { clear<kThreads>(zero, blockIdx.x, gridDim.x); }

// ---- gradient: sums of segments -------------------------------------------
//
// A segment is a table row's tokens of one window.  Its sum goes to the table
// (cleared before) where there is one window, else to the window's part of
// `parts`, and its byte of `named` is set.
//
// The sorted tokens are cut into chunks, one to a group of lanes.  The group in
// whose chunk a segment begins sums it to its end, in the next chunk too; only
// a segment that covers a whole chunk (which is then the first token of two
// chunks after each other, or begins with its chunk) is left in parts: the
// chunk it begins in writes tails[chunk], every further one heads[chunk], and
// k_segment_join adds them up.
//
// 6.55 million tokens of 128-byte rows take 79 us, 11 TB/s out of the chiplets'
// caches; vector instructions fill most of it (66 us: the additions, two tokens'
// packs at a time where no segment ends, a third of them).

struct Segments {
  uint32_t chunk, chunks;  // sorted tokens of a chunk, chunks of a window
  float *heads, *tails;    // [window][chunk][dim]
  float* parts;            // [window][vocabulary][dim], or null
  uint8_t* named;          // [window][vocabulary], with parts
  int64_t dim, stride;
  float scale;
};

template <typename T, int kSize>
__device__ __forceinline__ void store_segment(const Segments& g, T* out, uint32_t vocabulary, uint32_t window,
                                              uint32_t key, int64_t at, float* sum) {
  const uint64_t row = (uint64_t)window * vocabulary + key;
  if (g.parts) {
    Raw<float, kSize == 1 ? 1 : 4> v;
#pragma unroll
    for (int e = 0; e < kSize; e += kSize == 1 ? 1 : 4) v.put(sum + e, g.parts + row * g.dim + at + e);
    if (at == 0) g.named[row] = 1;
  } else {
#pragma unroll
    for (int e = 0; e < kSize; ++e) sum[e] *= g.scale;
    Raw<T, kSize>().put(sum, out + row * g.dim + at);
  }
}

template <int kSize>
__device__ __forceinline__ void store_floats(float* to, const float* sum) {
  Raw<float, kSize == 1 ? 1 : 4> v;
#pragma unroll
  for (int e = 0; e < kSize; e += kSize == 1 ? 1 : 4) v.put(sum + e, to + e);
}

template <int kSize>
__device__ __forceinline__ void add_floats(const float* from, float* sum) {
#pragma unroll
  for (int e = 0; e < kSize; e += kSize == 1 ? 1 : 4) {
    Raw<float, kSize == 1 ? 1 : 4> v;
    float x[4];
    v.load(from + e);
    v.get(x);
#pragma unroll
    for (int k = 0; k < (kSize == 1 ? 1 : 4); ++k) sum[e + k] += x[k];
  }
}

// Adds the rows first, first + step, .. below end of a matrix of floats, kAhead
// of them in flight.
template <int kSize>
__device__ __forceinline__ void add_rows(const float* matrix, int64_t dim, uint32_t first, uint32_t end, uint32_t step,
                                         float* sum) {
  constexpr int kPart = kSize == 1 ? 1 : 4;
  for (uint32_t r = first; r < end; r += kAhead * step) {
    Raw<float, kPart> v[kAhead][kSize / kPart];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t row = r + j * step < end ? r + j * step : r;
#pragma unroll
      for (int e = 0; e < kSize / kPart; ++e) v[j][e].load(matrix + (uint64_t)row * dim + e * kPart);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (r + j * step < end)
#pragma unroll
        for (int e = 0; e < kSize / kPart; ++e) {
          float x[kPart];
          v[j][e].get(x);
#pragma unroll
          for (int k = 0; k < kPart; ++k) sum[e * kPart + k] += x[k];
        }
  }
}

// Table rows by their place among a window's sorted entries.
template <typename E>
struct Keys {
  const E* entries;
  int row_bits;
  __device__ uint32_t operator()(uint32_t i) const { return (uint32_t)(entries[i] >> row_bits); }
};

// O: byte offsets into a window's rows of grad, 32 bits where those are less
// than 4 GB (30,000 x 300 tokens of 128 columns 265 us, with 64 bits 278).
template <typename T, typename E, typename O, int kLanes, int kSize>
__global__ __launch_bounds__(kThreads) void k_segment_sums(T* __restrict__ out, const T* __restrict__ grad,
                                                           const E* __restrict__ sorted, Sort s, Segments g) {
  constexpr uint32_t kGroups = kThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  uint32_t window, part;
  window_of(s.windows, (g.chunks + kGroups - 1) / kGroups, blockIdx.x, &window, &part);
  const uint32_t c = part * kGroups + threadIdx.x / kLanes, n = window_tokens(s, window);
  const uint64_t begin64 = (uint64_t)c * g.chunk;
  if (c >= g.chunks || begin64 >= n) return;
  int64_t at;
  const bool active = columns_of<kLanes, kSize>(lane, g.dim, &at);
  const uint32_t begin = (uint32_t)begin64, end = n - begin < g.chunk ? n : begin + g.chunk;
  const E* entries = sorted + (uint64_t)window * s.tokens;
  const Keys<E> key_at = {entries, s.row_bits};
  const char* rows = (const char*)(grad + (int64_t)window * s.window * g.stride);
  const O column = (O)(at * (int64_t)sizeof(T));
  const int64_t stride_bytes = g.stride * (int64_t)sizeof(T);
  const float one = runtime_one();
  const E mask = ((E)1 << s.row_bits) - 1;
  const uint32_t front = key_at(begin), back = key_at(end - 1);
  const uint32_t before = begin > 0 ? key_at(begin - 1) : ~0u;
  const uint32_t front_before = begin > 0 ? key_at(begin - g.chunk) : ~0u;
  const uint32_t after = end < n ? key_at(end) : ~0u;
  const uint32_t front_after = (uint64_t)end + g.chunk < n ? key_at(end + g.chunk) : ~0u;
  // The segment that reaches in from the chunk before: its owner sums it, or
  // it is one left in parts.
  bool head = before == front && (front_before == front || after == front);
  bool skip = before == front && !head;
  // The segment that reaches out: summed to its end, or left.
  const bool goes_on = after == back, own = !(before == front && front == back);
  const bool follow = goes_on && own && front != back && front_after != back;
  const uint32_t limit = !follow ? end : (n - end < g.chunk ? n : end + g.chunk);
  if (front >= s.vocabulary) return;
  uint32_t key = front, i = begin;
  if (skip)
    while (i + kAhead < end && key_at(i + kAhead) == front) i += kAhead;
  float sum[kSize] = {};
  // A lane's share of the next eight entries is fetched an iteration ahead, with
  // the entry behind each.
  constexpr int kMine = kShare<kLanes>;
  E mine[kMine], behind[kMine];
  auto fetch = [&](uint32_t from) {
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const uint32_t p = from + (kMine == 1 ? lane % kAhead : j);
      mine[j] = entries[p < n ? p : n - 1];
      behind[j] = p + 1 < n ? entries[p + 1] : ~(E)0;
    }
  };
  fetch(i);
  for (; i < limit; i += kAhead) {
    O offset[kMine];
    uint32_t after_each[kMine];  // the key behind each entry
    // Where something is to be done behind an entry: its segment ends, or the walk
    // does.  `mine_ends` has the eight of this lane's group, `any_ends` those of
    // any group of the wave.
    bool ends_here[kMine];
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      offset[j] = (O)((int64_t)(mine[j] & mask) * stride_bytes);
      after_each[j] = (uint32_t)(behind[j] >> s.row_bits);
      const uint32_t p = i + (kMine == 1 ? lane % kAhead : j) + 1;
      ends_here[j] = after_each[j] != (uint32_t)(mine[j] >> s.row_bits) || p >= n || p == end || p >= limit;
    }
    uint32_t mine_ends = 0, any_ends = 0;
    if constexpr (kMine == 1) {
      const uint64_t all = __ballot(ends_here[0]);
      mine_ends = (uint32_t)(all >> (lane_id() / kAhead * kAhead)) & 0xff;
      const uint32_t folded = (uint32_t)all | (uint32_t)(all >> 32);
      any_ends = (folded | folded >> 8 | folded >> 16 | folded >> 24) & 0xff;
    } else {
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        mine_ends |= (uint32_t)ends_here[j] << j;
        any_ends |= (uint32_t)__any(ends_here[j]) << j;
      }
    }
    fetch(i + kAhead);
    O from[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) from[j] = share_of<kLanes>(offset, j) + column;
    Raw<T, kSize> v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v[j].load((const T*)(rows + from[j]));
    bool done = false;
    auto behind_entry = [&](int j) {
      const uint32_t following = share_of<kLanes>(after_each, j);
      const uint32_t p = i + j + 1;  // the tokens up to here
      const bool ends = p >= n || following != key;
      if (mine_ends >> j & 1 && (ends || p != end || !follow)) {
        if (active && key < s.vocabulary && !skip) {
          if (ends && !head) {
            store_segment<T, kSize>(g, out, s.vocabulary, window, key, at, sum);
          } else {
            store_floats<kSize>((head ? g.heads : g.tails) + ((uint64_t)window * g.chunks + c) * g.dim + at, sum);
          }
        }
        if (p >= end || following >= s.vocabulary) {
          done = true;
          mine_ends = 0;
        }
        key = following;
        head = skip = false;
#pragma unroll
        for (int e = 0; e < kSize; ++e) sum[e] = 0.0f;
      }
    };
#pragma unroll
    for (int j = 0; j < kAhead; j += 2) {
      if (any_ends >> j & 1) {
        add_one<T, kSize>(v[j], one, sum);
        behind_entry(j);
        add_one<T, kSize>(v[j + 1], one, sum);
      } else {
        add_two<T, kSize>(v[j], v[j + 1], one, sum);
      }
      if (any_ends >> (j + 1) & 1) behind_entry(j + 1);
    }
    if (done) break;
  }
}

// Chunks of a workgroup of k_segment_join, and the heads from which on all its
// groups share a segment.
constexpr uint32_t kJoinChunks = 64, kJoinLong = 32;
constexpr int kJoinThreads = 256;

// Segments left in parts that begin in kJoinChunks chunks.
template <typename T, typename E, int kLanes, int kSize>
__global__ __launch_bounds__(kJoinThreads) void k_segment_join(T* __restrict__ out, const E* __restrict__ sorted, Sort s,
                                                           Segments g) {
  constexpr int kGroups = kJoinThreads / kLanes;
  __shared__ float shared[kJoinThreads * kSize];
  __shared__ uint32_t short_chunk[kJoinChunks], short_heads[kJoinChunks], long_chunk[kJoinChunks];
  __shared__ uint32_t shorts, longs, run;
  if (threadIdx.x == 0) shorts = longs = 0;
  __syncthreads();
  uint32_t window, part;
  window_of(s.windows, (g.chunks + kJoinChunks - 1) / kJoinChunks, blockIdx.x, &window, &part);
  const uint32_t n = window_tokens(s, window);
  const Keys<E> key_at = {sorted + (uint64_t)window * s.tokens, s.row_bits};
  const uint32_t first = part * kJoinChunks;
  if (threadIdx.x < kJoinChunks) {
    const uint32_t c = first + threadIdx.x;
    const uint64_t end64 = (uint64_t)(c + 1) * g.chunk;
    if (c < g.chunks && end64 < n) {
      const uint32_t end = (uint32_t)end64, begin = end - g.chunk, key = key_at(end);
      const uint32_t front = key_at(begin), before = begin > 0 ? key_at(begin - 1) : ~0u;
      const uint32_t front_after = (uint64_t)end + g.chunk < n ? key_at(end + g.chunk) : ~0u;
      if (key_at(end - 1) == key && key < s.vocabulary && !(front == key && before == key) &&
          (front == key || front_after == key)) {
        // The chunks that begin with its key: eight looked at together, then the others.
        uint32_t heads = 1;
        bool more = true;
        auto probe = [&](auto first, auto last) {
          uint32_t fronts[kJoinLong];
#pragma unroll
          for (uint32_t j = decltype(first)::value; j < decltype(last)::value; ++j) {
            const uint64_t i = (uint64_t)end + (uint64_t)j * g.chunk;
            fronts[j] = i < n ? key_at((uint32_t)i) : ~0u;
          }
#pragma unroll
          for (uint32_t j = decltype(first)::value; j < decltype(last)::value; ++j) {
            more = more && fronts[j] == key;
            heads += more;
          }
        };
        probe(std::integral_constant<uint32_t, 1>(), std::integral_constant<uint32_t, 8>());
        if (more) probe(std::integral_constant<uint32_t, 8>(), std::integral_constant<uint32_t, kJoinLong>());
        if (heads < kJoinLong) {  // (kJoinLong may not be all of them)
          const uint32_t k = atomicAdd(&shorts, 1u);
          short_chunk[k] = c;
          short_heads[k] = heads;
        } else {
          long_chunk[atomicAdd(&longs, 1u)] = c;
        }
      }
    }
  }
  __syncthreads();
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  int64_t at;
  const bool active = columns_of<kLanes, kSize>(lane, g.dim, &at);
  const uint64_t here = (uint64_t)window * g.chunks;
  for (uint32_t k = group; k < shorts; k += kGroups) {
    if (!active) break;
    const uint32_t c = short_chunk[k], key = key_at((c + 1) * g.chunk);
    float sum[kSize] = {};
    add_floats<kSize>(g.tails + (here + c) * g.dim + at, sum);
    add_rows<kSize>(g.heads + (here + c) * g.dim + at, g.dim, 1, 1 + short_heads[k], 1, sum);
    store_segment<T, kSize>(g, out, s.vocabulary, window, key, at, sum);
  }
  for (uint32_t k = 0; k < longs; ++k) {
    const uint32_t c = long_chunk[k], key = key_at((c + 1) * g.chunk);
    uint32_t heads = kJoinLong;
    for (;;) {
      if (threadIdx.x == 0) run = kJoinThreads;
      __syncthreads();
      const uint64_t i = (uint64_t)(c + 1 + heads + threadIdx.x) * g.chunk;
      if (i >= n || key_at((uint32_t)i) != key) atomicMin(&run, threadIdx.x);
      __syncthreads();
      const uint32_t more = run;
      __syncthreads();
      heads += more;
      if (more < kJoinThreads) break;
    }
    float sum[kSize] = {};
    if (active) add_rows<kSize>(g.heads + (here + c) * g.dim + at, g.dim, 1 + group, 1 + heads, kGroups, sum);
#pragma unroll
    for (int e = 0; e < kSize; ++e) shared[threadIdx.x * kSize + e] = sum[e];
    __syncthreads();
    if (group == 0 && active) {
#pragma unroll
      for (int e = 0; e < kSize; ++e) sum[e] = 0.0f;
      add_floats<kSize>(g.tails + (here + c) * g.dim + at, sum);
      for (int other = 0; other < kGroups; ++other)
#pragma unroll
        for (int e = 0; e < kSize; ++e) sum[e] += shared[(lane + other * kLanes) * kSize + e];
      store_segment<T, kSize>(g, out, s.vocabulary, window, key, at, sum);
    }
    __syncthreads();
  }
}

// ---- gradient: few tokens, in one launch ------------------------------------
//
// Workgroup w has `range` rows of the table.  It reads all tokens, a wave a
// sixteenth of them in their order, keeps those of its rows, sorts them and sums
// their segments; its rows that no token names become zero.  Reading all tokens
// 256 times from cache costs less than the launches between sorting and summing:
// 256 x 100 tokens, 12.5 us; in five launches, 27.

constexpr int kRangeThreads = 1024, kRangeWaves = kRangeThreads / kWave;
constexpr uint32_t kRanges = 256;  // workgroups at most, and table rows of each at most

template <typename T, typename I, int kLanes, int kSize>
__global__ __launch_bounds__(kRangeThreads) void k_range_gradient(T* __restrict__ out, uint32_t* __restrict__ sorted,
                                                                  const T* __restrict__ grad,
                                                                  const I* __restrict__ tokens, Sort s, int64_t dim,
                                                                  int64_t stride, float scale, uint32_t range,
                                                                  uint32_t share) {
  constexpr uint32_t kGroups = kRangeThreads / kLanes;
  extern __shared__ __align__(16) uint8_t lds[];
  uint32_t(*counts)[kDigits] = (uint32_t(*)[kDigits])lds;  // [wave][table row]
  uint32_t* totals = (uint32_t*)(counts + kRangeWaves);
  uint32_t* shared = totals + kDigits;
  uint32_t* smaller = shared + 2 * kRangeWaves;            // tokens of rows below, by wave
  uint32_t* room = smaller + kRangeWaves;                  // the waves' tokens, then the groups' heads
  const uint32_t lane = lane_id(), wave = threadIdx.x / kWave, n = (uint32_t)s.tokens;
  const uint32_t low = blockIdx.x * range;
  range = s.vocabulary - low < range ? s.vocabulary - low : range;
  uint32_t* mine = room + wave * share;
  for (uint32_t d = lane; d < kDigits; d += kWave) counts[wave][d] = 0;
  const uint32_t begin = wave * share, end = begin + share < n ? begin + share : n;
  uint32_t found = 0, before = 0;
  for (uint32_t first = begin; first < end; first += kAhead * kWave) {
    // A token's low word is compared; those outside the table lie above every row.
    uint32_t key[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t i = first + j * kWave + lane;
      const I id = i < end ? tokens[i] : I(-1);
      if constexpr (sizeof(I) == 8) key[j] = (uint64_t)id >> 31 ? ~0u : (uint32_t)id;
      else key[j] = (uint32_t)id;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const bool in = key[j] - low < range;
      const uint64_t all = __ballot(in);
      before += (uint32_t)__popcll(__ballot(key[j] < low));
      if (all == 0) continue;
      if (in) {
        const uint32_t i = first + j * kWave + lane;
        mine[found + (uint32_t)__popcll(all & ((1ull << lane) - 1))] = key[j] << s.row_bits | i / s.bag;
        atomicAdd(&counts[wave][key[j] - low], 1u);
      }
      found += (uint32_t)__popcll(all);
    }
  }
  if (lane == 0) smaller[wave] = before;
  __syncthreads();
  // A table row's tokens wave by wave, after the rows below it and the ranges below.
  if (threadIdx.x < kDigits) {
    uint32_t offset = 0;
#pragma unroll
    for (int w = 0; w < kRangeWaves; ++w) {
      const uint32_t c = counts[w][threadIdx.x];
      counts[w][threadIdx.x] = offset;
      offset += c;
    }
    totals[threadIdx.x] = offset;
  }
  __syncthreads();
  scan_digits(totals, shared);
  uint32_t start = 0;
#pragma unroll
  for (int w = 0; w < kRangeWaves; ++w) start += smaller[w];
  uint32_t* entries = sorted + start;
  for (uint32_t first = 0; first < found; first += kWave) {
    const bool valid = first + lane < found;
    const uint32_t entry = valid ? mine[first + lane] : 0, digit = valid ? (entry >> s.row_bits) - low : 0;
    const uint64_t same = equal_digits(digit, __ballot(valid));
    const int leader = same ? __ffsll((unsigned long long)same) - 1 : (int)lane;
    uint32_t at = 0;
    if (valid && leader == (int)lane) at = atomicAdd(&counts[wave][digit], (uint32_t)__popcll(same));
    at = __shfl(at, leader, kWave);
    if (valid) entries[totals[digit] + at + (uint32_t)__popcll(same & ((1ull << lane) - 1))] = entry;
  }
  __syncthreads();
  const uint32_t c = totals[kDigits - 1];  // all of them: no row is the last digit
  // Sums.  A group of lanes takes `chunk` sorted tokens; what belongs to a segment of
  // the chunk before goes to its head, and the group in whose chunk a segment begins
  // adds the heads it runs through.
  const uint32_t lane_in = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const uint32_t chunk = ((c + kGroups - 1) / kGroups + kAhead - 1) / kAhead * kAhead;
  const uint32_t from = group * chunk < c ? group * chunk : c, to = c - from < chunk ? c : from + chunk;
  const uint32_t mask = (1u << s.row_bits) - 1;
  float* heads = (float*)room;
  uint32_t* fronts = (uint32_t*)(heads + kRangeThreads * kSize);  // each group's first key, ~0 without tokens
  if (lane_in == 0) fronts[group] = from < to ? entries[from] >> s.row_bits : ~0u;
  const float one = runtime_one();
  // (The groups that take this path have all columns of a row at once.)
  const int64_t nominal = lane_in * kSize, at = nominal < dim - kSize ? nominal : dim - kSize;
  const bool active = nominal < dim;
  float sum[kSize] = {};
  auto store = [&](uint32_t key) {
    if (!active) return;
#pragma unroll
    for (int e = 0; e < kSize; ++e) sum[e] *= scale;
    Raw<T, kSize>().put(sum, out + (int64_t)key * dim + at);
  };
  bool head = from > 0 && from < to && entries[from - 1] >> s.row_bits == entries[from] >> s.row_bits, tail = false;
  uint32_t key = from < to ? entries[from] >> s.row_bits : 0;
  // Entries are fetched an iteration ahead, with the one behind them.
  uint32_t next[kAhead + 1];
  auto fetch = [&](uint32_t i) {
#pragma unroll
    for (int j = 0; j <= kAhead; ++j) next[j] = entries[i + j < c ? i + j : c - 1];
  };
  if (from < to) fetch(from);
  for (uint32_t i = from; i < to; i += kAhead) {
    uint32_t entry[kAhead + 1];
#pragma unroll
    for (int j = 0; j <= kAhead; ++j) entry[j] = next[j];
    if (i + kAhead < to) fetch(i + kAhead);
    Raw<T, kSize> v[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v[j].load(grad + (int64_t)(entry[j] & mask) * stride + at);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t p = i + j + 1;
      if (p > to) break;
      add_one<T, kSize>(v[j], one, sum);
      const uint32_t following = entry[j + 1] >> s.row_bits;
      const bool ends = p >= c || following != key;
      if (!ends && p < to) continue;
      if (head) store_floats<kSize>(heads + (size_t)threadIdx.x * kSize, sum);
      else if (ends) store(key);
      else tail = true;
      if (tail) break;
      key = following;
      head = false;
#pragma unroll
      for (int e = 0; e < kSize; ++e) sum[e] = 0.0f;
    }
  }
  __syncthreads();
  if (tail) {
    for (uint32_t g = group + 1; g < kGroups && fronts[g] == key; ++g)
      add_floats<kSize>(heads + (size_t)(g * kLanes + lane_in) * kSize, sum);
    store(key);
  }
  // Rows without tokens.
  for (uint32_t r = group; r < range; r += kGroups)
    if (totals[r] == totals[r + 1]) {
#pragma unroll
      for (int e = 0; e < kSize; ++e) sum[e] = 0.0f;
      store(low + r);
    }
}

// The table from its windows' parts.
template <typename T, int kLanes, int kSize>
__global__ __launch_bounds__(kThreads) void k_segment_windows(T* __restrict__ out, uint32_t vocabulary,
                                                              uint32_t windows, Segments g) {
  constexpr uint32_t kGroups = kThreads / kLanes;
  int64_t at;
  if (!columns_of<kLanes, kSize>(threadIdx.x % kLanes, g.dim, &at)) return;
  for (uint64_t row = (uint64_t)blockIdx.x * kGroups + threadIdx.x / kLanes; row < vocabulary;
       row += (uint64_t)gridDim.x * kGroups) {
    float sum[kSize] = {};
    for (uint32_t w = 0; w < windows; ++w) {
      const uint64_t from = (uint64_t)w * vocabulary + row;
      if (g.named[from]) add_floats<kSize>(g.parts + from * g.dim + at, sum);
    }
#pragma unroll
    for (int e = 0; e < kSize; ++e) sum[e] *= g.scale;
    Raw<T, kSize>().put(sum, out + row * g.dim + at);
  }
}

// ---- host -------------------------------------------------------------------

// Lanes that share a row, a power of two up to a wave, and the columns of each.
struct RowLanes {
  int lanes, size;
  int64_t groups;  // of lanes, side by side in a row
};

RowLanes row_lanes(int64_t dim, int pack) {
  RowLanes r = {1, dim < pack ? 1 : pack, 0};
  const int64_t packs = (dim + r.size - 1) / r.size;
  while (r.lanes < kWave && r.lanes < packs) r.lanes *= 2;
  r.groups = (packs + r.lanes - 1) / r.lanes;
  return r;
}

// fn(lanes, columns of a lane) with both as constants.
template <typename T, typename F>
void with_lanes(const RowLanes& r, F&& fn) {
  constexpr int kPack = Pack<T>::kSize;
  using One = std::integral_constant<int, 1>;
  using Full = std::integral_constant<int, kPack>;
  if (r.size == 1) {
    switch (r.lanes) {
      case 1: fn(One(), One()); break;
      case 2: fn(std::integral_constant<int, 2>(), One()); break;
      case 4: fn(std::integral_constant<int, 4>(), One()); break;
      default: fn(std::integral_constant<int, 8>(), One()); break;
    }
    return;
  }
  switch (r.lanes) {
    case 1: fn(One(), Full()); break;
    case 2: fn(std::integral_constant<int, 2>(), Full()); break;
    case 4: fn(std::integral_constant<int, 4>(), Full()); break;
    case 8: fn(std::integral_constant<int, 8>(), Full()); break;
    case 16: fn(std::integral_constant<int, 16>(), Full()); break;
    case 32: fn(std::integral_constant<int, 32>(), Full()); break;
    default: fn(std::integral_constant<int, 64>(), Full()); break;
  }
}

// Lanes that keep the chip's memory busy: four waves on each SIMD of 256 CUs.
// Groups share a row's tokens below that (us, shared and a group a row): 16 x 100
// tokens of 32 columns 3.4 and 9.2, 2,000 x 100 of 64 columns 6.9 and 10.2, 20,000 x 100
// 21.7 and 21.1.
constexpr int64_t kBusyLanes = int64_t(1) << 18;

template <typename T, typename I>
int lookup(T* out, const T* weight, const I* tokens, int64_t rows, int64_t bag, int64_t vocabulary, int64_t dim,
           int64_t stride, float scale, hipStream_t stream) {
  const RowLanes r = row_lanes(dim, Pack<T>::kSize);
  // Few rows: groups share a row's tokens until the chip is busy.
  int split = 1;
  while (split * 2 * r.lanes <= kThreads && rows * r.groups * r.lanes * split < kBusyLanes &&
         (int64_t)split * kAhead < bag)
    split *= 2;
  const int rows_here = kThreads / r.lanes / split;
  const int64_t wanted = (rows + rows_here - 1) / rows_here;
  const dim3 grid((uint32_t)(wanted < (1 << 20) ? wanted : (1 << 20)), (uint32_t)r.groups);
  const int64_t stride_bytes = stride * (int64_t)sizeof(T), table = stride_bytes * vocabulary + dim * (int64_t)sizeof(T);
  const bool near = stride >= 0 && table < (int64_t(1) << 32);
  with_lanes<T>(r, [&](auto l, auto s) {
    constexpr int kLanes = decltype(l)::value, kSize = decltype(s)::value;
    if (bag <= 1)
      hipLaunchKernelGGL((k_lookup<T, I, kLanes, kSize>), grid, dim3(kThreads), 0, stream, out, weight, tokens, rows,
                         bag, vocabulary, dim, stride, scale);
    else if (near)
      hipLaunchKernelGGL((k_lookup_pooled<T, I, uint32_t, kLanes, kSize>), grid, dim3(kThreads), 0, stream, out, weight,
                         tokens, rows, bag, (uint32_t)vocabulary, dim, stride_bytes, scale, split);
    else
      hipLaunchKernelGGL((k_lookup_pooled<T, I, int64_t, kLanes, kSize>), grid, dim3(kThreads), 0, stream, out, weight,
                         tokens, rows, bag, (uint32_t)vocabulary, dim, stride_bytes, scale, split);
  });
  MGB_LAUNCH_CHECK("embedding lookup");
  return 0;
}

// A chiplet's cache, and the part of it that a window's rows of grad may take.  us
// with one window, and with windows of 1, 2.25 and 4 MB: 65,536 x 100 tokens of 128
// bytes 214, 180, 182, 191; 131,072 x 100 of 128 bytes 365, 269, 264, 279; 262,144 x 50
// of 256 bytes 675, 619, 518, 452.
constexpr int64_t kCache = int64_t(4) << 20, kWindowBytes = int64_t(9) << 18;
// Most tokens for the one launch by ranges (LDS holds them all, were they one range's).
// At 32,700 tokens 13.3 us, sorted in three launches 25.5 (32 columns); 17.0 and 29.1
// (256 columns).
constexpr int64_t kRangeTokens = 32768;
// Tokens from which a tile has 16 rounds, not 4 (us, 4 and 16): 1 million tokens of 64
// columns 70 and 82, 3 million of 32 columns 117 and 118, 10 million of 16 columns 282
// and 273.
constexpr int64_t kLongTiles = int64_t(1) << 21;
// Sorted tokens of a group at most (us, 64, 128, 512 and 2,048): 65,536 x 100 tokens of
// 64 columns 191, 181, 182, 182; 262,144 x 50 of 128 columns 472, 454, 516, 517.
constexpr int64_t kMostChunk = 512;

// How the gradient of rows x bag tokens is computed and laid out in the workspace.
struct GradientPlan {
  Sort sort;
  Segments segments;
  RowLanes row;
  bool wide, by_range, few;  // 64-bit entries; one launch by ranges; few tiles
  int passes, rounds;
  size_t entries[2], counts, totals, heads, tails, parts, named, next_counts, clear_bytes, bytes;
};

int bits_of(uint64_t v) {
  int bits = 0;
  while (v >> bits) ++bits;
  return bits;
}

GradientPlan gradient_plan(int64_t rows, int64_t bag, int64_t vocabulary, int64_t dim, int size) {
  GradientPlan p = {};
  const int64_t n = rows * bag;
  p.row = row_lanes(dim, size);
  // Windows that a chiplet's cache holds, where a table row keeps at least 16
  // tokens in each: its partial sums are then few against what they gather.
  int64_t windows = 1;
  const int64_t bytes = rows * dim * (16 / size), most = n / (16 * vocabulary);
  if (bytes > kCache)
    while (windows * kWindowBytes < bytes && (windows < kChiplets ? 2 * windows : windows + kChiplets) <= most)
      windows = windows < kChiplets ? 2 * windows : windows + kChiplets;
  const int64_t window = (rows + windows - 1) / windows;
  const int key_bits = bits_of(vocabulary), row_bits = bits_of(window - 1);
  p.passes = (key_bits + kDigitBits - 1) / kDigitBits;
  p.wide = key_bits + row_bits > 32;
  p.by_range = windows == 1 && !p.wide && n <= kRangeTokens && vocabulary < kRanges * (kDigits - 1) && p.row.groups == 1;
  p.few = !p.by_range && windows == 1 && n <= (int64_t)kFewTiles * 4 * kSortThreads;
  p.rounds = p.few ? 1 : n < kLongTiles ? 4 : 16;
  while (p.few && n > (int64_t)kFewTiles * p.rounds * kSortThreads) p.rounds *= 2;
  const int64_t tile = (int64_t)p.rounds * kSortThreads;
  p.sort.vocabulary = (uint32_t)vocabulary;
  p.sort.bag = (uint32_t)bag;
  p.sort.rows = (uint32_t)rows;
  p.sort.window = (uint32_t)window;
  p.sort.windows = (uint32_t)windows;
  p.sort.tiles = (uint32_t)((window * bag + tile - 1) / tile);
  p.sort.row_bits = row_bits;
  p.sort.digit_bits = (key_bits + p.passes - 1) / p.passes;
  p.sort.tokens = (uint64_t)(window * bag);
  // Sorted tokens of a group: enough groups for the chip, then longer walks,
  // which leave fewer parts to join.
  int64_t chunk = n * p.row.lanes * p.row.groups / (2 * kBusyLanes);
  chunk = (chunk + kAhead - 1) / kAhead * kAhead;
  chunk = chunk < kAhead ? kAhead : chunk > kMostChunk ? kMostChunk : chunk;
  p.segments.chunk = (uint32_t)chunk;
  p.segments.chunks = (uint32_t)((window * bag + chunk - 1) / chunk);
  p.segments.dim = dim;
  size_t at = 0;
  auto take = [&](size_t want) {
    const size_t from = at;
    at += (want + 255) / 256 * 256;
    return from;
  };
  const size_t sorted = (size_t)n * (p.wide ? 8 : 4);
  p.entries[0] = take(sorted);
  p.entries[1] = p.by_range ? p.entries[0] : take(sorted);
  if (!p.by_range) {
    p.counts = take((size_t)windows * kDigits * p.sort.tiles * sizeof(uint32_t));
    p.totals = take((size_t)windows * kDigits * sizeof(uint32_t));
  }
  if (p.by_range) {
    p.bytes = at;
    return p;
  }
  p.heads = take((size_t)windows * p.segments.chunks * dim * sizeof(float));
  p.tails = take((size_t)windows * p.segments.chunks * dim * sizeof(float));
  if (windows > 1) p.parts = take((size_t)windows * vocabulary * dim * sizeof(float));
  // Cleared together: the rows' bytes or the later passes' counts.
  p.clear_bytes = windows > 1 ? (size_t)windows * vocabulary
                              : p.few ? (size_t)(p.passes - 1) * p.sort.tiles * kDigits * sizeof(uint32_t) : 0;
  p.named = p.next_counts = take(p.clear_bytes);
  p.bytes = at;
  return p;
}

uint32_t at_most(uint64_t wanted, uint32_t most) { return wanted < most ? (uint32_t)wanted : most; }

// What the sort's launches clear: the first the workspace's part, each a share
// of the table.
struct Clearing {
  Clear first;     // [0]: the workspace
  uint8_t* table;
  uint64_t left;
  int launches;    // still to come
};

Clear next_clear(Clearing& c) {
  Clear now = c.first;
  c.first = {};
  const uint64_t share = c.launches > 1 ? c.left / c.launches / 256 * 256 : c.left;
  now.at[1] = c.table;
  now.bytes[1] = share;
  c.table += share;
  c.left -= share;
  --c.launches;
  return now;
}

// Workgroups for it: 128 bytes a lane.
uint32_t clear_blocks(const Clear& c, int threads) {
  const uint64_t bytes = c.bytes[0] > c.bytes[1] ? c.bytes[0] : c.bytes[1];
  return at_most((bytes + 128 * threads - 1) / (128 * threads), 1024);
}

template <typename E, typename F, int kRounds, bool kFew>
void sort_pass(const GradientPlan& p, uint8_t* ws, F from, E* out, int pass, Clearing& clearing, hipStream_t stream) {
  uint32_t *counts = (uint32_t*)(ws + p.counts), *totals = (uint32_t*)(ws + p.totals);
  uint32_t* later = (uint32_t*)(ws + p.next_counts);  // [pass - 1][tile][digit]
  const uint32_t blocks = p.sort.windows * p.sort.tiles, each = p.sort.tiles * kDigits;
  if (pass == 0 || !kFew) {
    const Clear zero = next_clear(clearing);
    hipLaunchKernelGGL((k_sort_count<F, kRounds, kFew>), dim3(blocks + clear_blocks(zero, kSortThreads)),
                       dim3(kSortThreads), 0, stream, counts, from, p.sort, pass, zero);
  }
  if (!kFew)
    hipLaunchKernelGGL(k_sort_scan, dim3(p.sort.windows * kDigits), dim3(kThreads), 0, stream, counts, totals,
                       p.sort.tiles);
  if (kFew && pass > 0) counts = later + (size_t)(pass - 1) * each;
  const Clear zero = next_clear(clearing);
  hipLaunchKernelGGL((k_sort_scatter<E, F, kRounds, kFew>), dim3(blocks + clear_blocks(zero, kSortThreads)),
                     dim3(kSortThreads), 0, stream, out, from, counts, totals,
                     kFew && pass + 1 < p.passes ? later + (size_t)pass * each : nullptr, p.sort, pass, zero);
}

// The sorted entries' place.
template <typename E, typename I>
E* sort_tokens(const GradientPlan& p, uint8_t* ws, const I* tokens, Clearing clearing, hipStream_t stream) {
  E* entries[2] = {(E*)(ws + p.entries[0]), (E*)(ws + p.entries[1])};
  clearing.launches = p.few ? p.passes + 1 : 2 * p.passes;
  int now = 0;
  for (int pass = 0; pass < p.passes; ++pass, now ^= 1) {
    auto run = [&](auto from) {
      using F = decltype(from);
      if (p.few) {
        if (p.rounds == 1) sort_pass<E, F, 1, true>(p, ws, from, entries[now], pass, clearing, stream);
        else if (p.rounds == 2) sort_pass<E, F, 2, true>(p, ws, from, entries[now], pass, clearing, stream);
        else sort_pass<E, F, 4, true>(p, ws, from, entries[now], pass, clearing, stream);
      } else if (p.rounds == 4) {
        sort_pass<E, F, 4, false>(p, ws, from, entries[now], pass, clearing, stream);
      } else {
        sort_pass<E, F, 16, false>(p, ws, from, entries[now], pass, clearing, stream);
      }
    };
    if (pass == 0) run(TokenEntries<E, I>{tokens});
    else run(SortedEntries<E>{entries[now ^ 1]});
  }
  return entries[now ^ 1];
}

template <typename T, typename I>
int range_gradient(const GradientPlan& p, T* out, const T* grad, const I* tokens, uint8_t* ws, hipStream_t stream) {
  const uint32_t rows = p.sort.vocabulary, range = (rows + kRanges - 1) / kRanges, ranges = (rows + range - 1) / range;
  const uint32_t n = (uint32_t)p.sort.tokens, share = (n + kRangeThreads - 1) / kRangeThreads * kWave;
  int status = 0;
  with_lanes<T>(p.row, [&](auto l, auto size) {
    constexpr int kLanes = decltype(l)::value, kSize = decltype(size)::value;
    uint32_t room = kRangeWaves * share * 4;
    const uint32_t sums = (kRangeThreads * kSize + kRangeThreads / kLanes) * 4;
    if (room < sums) room = sums;
    const uint32_t lds = (kRangeWaves * kDigits + kDigits + 3 * kRangeWaves) * 4 + room;
    if (lds > 65536)
      status = check(hipFuncSetAttribute((const void*)k_range_gradient<T, I, kLanes, kSize>,
                                         hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds),
                     "hipFuncSetAttribute(k_range_gradient)");
    if (status == 0)
      hipLaunchKernelGGL((k_range_gradient<T, I, kLanes, kSize>), dim3(ranges), dim3(kRangeThreads), lds, stream, out,
                         (uint32_t*)(ws + p.entries[0]), grad, tokens, p.sort, p.segments.dim, p.segments.stride,
                         p.segments.scale, range, share);
  });
  if (status) return -1;
  MGB_LAUNCH_CHECK("embedding gradient: ranges");
  return 0;
}

template <typename T, typename E, typename I>
int lookup_gradient(GradientPlan& p, T* out, const T* grad, const I* tokens, uint8_t* ws, hipStream_t stream) {
  Clearing clearing = {};
  clearing.first.at[0] = ws + p.named;
  clearing.first.bytes[0] = p.clear_bytes;
  if (p.sort.windows == 1) {
    clearing.table = (uint8_t*)out;
    clearing.left = (uint64_t)p.sort.vocabulary * p.segments.dim * sizeof(T);
  }
  const E* sorted = sort_tokens<E, I>(p, ws, tokens, clearing, stream);
  MGB_LAUNCH_CHECK("embedding gradient: sort");
  with_lanes<T>(p.row, [&](auto l, auto size) {
    constexpr int kLanes = decltype(l)::value, kSize = decltype(size)::value;
    constexpr uint32_t kGroups = kThreads / kLanes;
    const uint32_t columns = (uint32_t)p.row.groups, windows = p.sort.windows, chunks = p.segments.chunks;
    const dim3 groups(windows * ((chunks + kGroups - 1) / kGroups), columns);
    const int64_t stride = p.segments.stride, reach = (stride * p.sort.window + p.segments.dim) * (int64_t)sizeof(T);
    if (stride >= 0 && reach < (int64_t(1) << 32))
      hipLaunchKernelGGL((k_segment_sums<T, E, uint32_t, kLanes, kSize>), groups, dim3(kThreads), 0, stream, out, grad,
                         sorted, p.sort, p.segments);
    else
      hipLaunchKernelGGL((k_segment_sums<T, E, int64_t, kLanes, kSize>), groups, dim3(kThreads), 0, stream, out, grad,
                         sorted, p.sort, p.segments);
    if (chunks > 1)
      hipLaunchKernelGGL((k_segment_join<T, E, kLanes, kSize>),
                         dim3(windows * ((chunks + kJoinChunks - 1) / kJoinChunks), columns), dim3(kJoinThreads), 0,
                         stream, out, sorted, p.sort, p.segments);
    if (windows > 1)
      hipLaunchKernelGGL((k_segment_windows<T, kLanes, kSize>),
                         dim3(at_most((p.sort.vocabulary + kGroups - 1) / kGroups, 4096), columns), dim3(kThreads), 0,
                         stream, out, p.sort.vocabulary, windows, p.segments);
  });
  MGB_LAUNCH_CHECK("embedding gradient: sums");
  return 0;
}

template <typename T, typename I>
int lookup_gradient(T* out, const T* grad, const I* tokens, int64_t rows, int64_t bag, int64_t vocabulary, int64_t dim,
                    int64_t stride, float scale, uint8_t* ws, hipStream_t stream) {
  constexpr int kSize = Pack<T>::kSize;
  if (rows * bag == 0) {
    Clear zero = {};
    zero.at[1] = (uint8_t*)out;
    zero.bytes[1] = (uint64_t)vocabulary * dim * sizeof(T);
    hipLaunchKernelGGL(k_clear, dim3(clear_blocks(zero, kThreads)), dim3(kThreads), 0, stream, zero);
    MGB_LAUNCH_CHECK("embedding gradient: clearing");
    return 0;
  }
  GradientPlan p = gradient_plan(rows, bag, vocabulary, dim, kSize);
  p.segments.heads = (float*)(ws + p.heads);
  p.segments.tails = (float*)(ws + p.tails);
  p.segments.parts = p.sort.windows > 1 ? (float*)(ws + p.parts) : nullptr;
  p.segments.named = p.sort.windows > 1 ? ws + p.named : nullptr;
  p.segments.stride = stride;
  p.segments.scale = scale;
  if (p.by_range) return range_gradient<T, I>(p, out, grad, tokens, ws, stream);
  return p.wide ? lookup_gradient<T, uint64_t, I>(p, out, grad, tokens, ws, stream)
                : lookup_gradient<T, uint32_t, I>(p, out, grad, tokens, ws, stream);
}

template <typename F>
int with_types(int dtype, int token_bytes, F&& fn) {
  MGB_REQUIRE(token_bytes == 4 || token_bytes == 8, "embedding: tokens must be int32 or int64");
  auto tokens = [&](auto* t) { return token_bytes == 4 ? fn(t, (int32_t*)nullptr) : fn(t, (int64_t*)nullptr); };
  switch (dtype) {
    case MGB_F32: return tokens((float*)nullptr);
    case MGB_F16: return tokens((_Float16*)nullptr);
    case MGB_BF16: return tokens((__bf16*)nullptr);
  }
  set_error("embedding: types must be float32, float16 or bfloat16");
  return -1;
}

constexpr int64_t kMost = (int64_t(1) << 31) - 1;

int check_sizes(int64_t rows, int64_t bag, int64_t vocabulary, int64_t dim, int64_t stride) {
  MGB_REQUIRE(rows >= 0 && bag >= 0 && rows <= (int64_t(1) << 40) && bag <= kMost, "embedding: sizes out of range");
  MGB_REQUIRE(bag == 0 || rows <= (int64_t(1) << 60) / bag, "embedding: sizes out of range");
  MGB_REQUIRE(vocabulary >= 1 && vocabulary <= kMost, "embedding: the table must have 1 to 2^31 - 1 rows");
  MGB_REQUIRE(dim >= 1 && dim <= (int64_t(1) << 22), "embedding: a row must have 1 to 2^22 values");
  MGB_REQUIRE(stride > -(int64_t(1) << 31) && stride < (int64_t(1) << 31), "embedding: row stride out of range");
  return 0;
}

}  // namespace
}  // namespace mgb

using namespace mgb;

extern "C" {

int mgb_embedding_lookup(void* out, const void* weight, const void* tokens, int64_t rows, int64_t bag,
                         int64_t vocabulary, int64_t dim, int64_t stride, float scale, int dtype, int token_bytes,
                         void* stream) {
  if (check_sizes(rows, bag, vocabulary, dim, stride)) return -1;
  if (rows == 0) return 0;
  MGB_REQUIRE(out && weight && (tokens || bag == 0), "embedding lookup: null pointer");
  return with_types(dtype, token_bytes, [&](auto* t, auto* i) {
    using T = std::remove_pointer_t<decltype(t)>;
    using I = std::remove_pointer_t<decltype(i)>;
    return lookup<T, I>((T*)out, (const T*)weight, (const I*)tokens, rows, bag, vocabulary, dim, stride, scale,
                        (hipStream_t)stream);
  });
}

size_t mgb_embedding_gradient_workspace_bytes(int64_t rows, int64_t bag, int64_t vocabulary, int64_t dim, int dtype) {
  if (rows < 1 || bag < 1 || bag > kMost || rows > kMost / bag || vocabulary < 1 || vocabulary > kMost || dim < 1)
    return 0;
  return gradient_plan(rows, bag, vocabulary, dim, dtype == MGB_F32 ? 4 : 8).bytes;
}

int mgb_embedding_gradient(void* out, const void* grad, const void* tokens, int64_t rows, int64_t bag,
                           int64_t vocabulary, int64_t dim, int64_t stride, float scale, int dtype, int token_bytes,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (check_sizes(rows, bag, vocabulary, dim, stride)) return -1;
  MGB_REQUIRE(bag == 0 || rows <= kMost / bag, "embedding gradient: tokens must be below 2^31");
  const int64_t count = rows * bag;
  MGB_REQUIRE(out && (count == 0 || (grad && tokens && workspace)), "embedding gradient: null pointer");
  MGB_REQUIRE(workspace_bytes >= mgb_embedding_gradient_workspace_bytes(rows, bag, vocabulary, dim, dtype),
              "embedding gradient: workspace too small");
  return with_types(dtype, token_bytes, [&](auto* t, auto* i) {
    using T = std::remove_pointer_t<decltype(t)>;
    using I = std::remove_pointer_t<decltype(i)>;
    return lookup_gradient<T, I>((T*)out, (const T*)grad, (const I*)tokens, rows, bag, vocabulary, dim, stride, scale,
                                 (uint8_t*)workspace, (hipStream_t)stream);
  });
}

}  // extern "C"
