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
#include <type_traits>

#include "encoder_common.hpp"

namespace mgb {
namespace {

constexpr int kThreads = 256;

// ---- lookup ---------------------------------------------------------------

// Tokens a lane has in flight at once.
constexpr int kAhead = 8;

// kLanes lanes hold a pack of a row's columns each (further columns are other
// workgroups', blockIdx.y); `split` groups share a row's tokens, kAhead in
// turn, and are joined through LDS in their order.
template <typename T, typename I, int kLanes, bool kPool>
__global__ __launch_bounds__(kThreads) void k_lookup(T* __restrict__ out, const T* __restrict__ weight,
                                                     const I* __restrict__ tokens, int64_t rows, int64_t bag,
                                                     int64_t vocabulary, int64_t dim, int64_t stride, float scale,
                                                     int split) {
  constexpr int kSize = Pack<T>::kSize;
  constexpr int kAt = kPool ? kAhead : 1;
  __shared__ float shared[kPool ? kThreads * kSize : 1];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int part = group % split, rows_here = kThreads / kLanes / split;
  const int64_t at = ((int64_t)blockIdx.y * kLanes + lane) * kSize;
  for (int64_t base = (int64_t)blockIdx.x * rows_here; base < rows; base += (int64_t)gridDim.x * rows_here) {
    const int64_t row = base + group / split;
    float sum[kSize] = {};
    if (row < rows) {
      for (int64_t first = (int64_t)part * kAt; first < bag; first += (int64_t)split * kAt) {
        const I* ids = tokens + row * bag + first;
        float v[kAt][kSize];
        bool present[kAt];
#pragma unroll
        for (int j = 0; j < kAt; ++j) {
          const int64_t id = first + j < bag ? (int64_t)ids[j] : -1;
          present[j] = id >= 0 && id < vocabulary;
          load_pack(weight + (present[j] ? id : 0) * stride, at, dim, v[j]);
        }
#pragma unroll
        for (int j = 0; j < kAt; ++j)
#pragma unroll
          for (int e = 0; e < kSize; ++e) sum[e] += present[j] ? v[j][e] : 0.0f;
      }
    }
    if constexpr (kPool) {
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
    }
    if (part == 0 && row < rows) {
#pragma unroll
      for (int e = 0; e < kSize; ++e) sum[e] *= scale;
      store_pack(out + row * dim, at, dim, sum);
    }
  }
}

// ---- gradient: stable radix sort of (token, row) ---------------------------

constexpr int kDigitBits = 8, kDigits = 1 << kDigitBits;
constexpr int kSortRounds = 16;                     // keys of a lane
constexpr int kSortTile = kThreads * kSortRounds;   // keys of a workgroup
constexpr int kSortWaves = kThreads / kWave;

// The table row of token i; `vocabulary`, beyond every row, for none.
template <typename I>
__device__ __forceinline__ uint32_t token_key(const I* tokens, int64_t i, uint32_t vocabulary) {
  const int64_t id = (int64_t)tokens[i];
  return id >= 0 && id < (int64_t)vocabulary ? (uint32_t)id : vocabulary;
}

// Keys of the first pass come from the tokens, of later ones from the pass before.
template <typename I>
struct TokenKeys {
  const I* tokens;
  uint32_t vocabulary, bag;
  __device__ uint32_t key(uint32_t i) const { return token_key(tokens, i, vocabulary); }
  __device__ uint32_t row(uint32_t i) const { return i / bag; }
};
struct SortedKeys {
  const uint32_t *keys, *rows;
  __device__ uint32_t key(uint32_t i) const { return keys[i]; }
  __device__ uint32_t row(uint32_t i) const { return rows[i]; }
};

// counts[digit][tile]
template <typename K>
__global__ __launch_bounds__(kThreads) void k_sort_count(uint32_t* __restrict__ counts, K keys, uint32_t n, int shift,
                                                         uint32_t mask, uint32_t tiles) {
  __shared__ uint32_t count[kDigits];
  count[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t first = blockIdx.x * kSortTile;
#pragma unroll
  for (int k = 0; k < kSortRounds; ++k) {
    const uint32_t i = first + k * kThreads + threadIdx.x;
    if (i < n) atomicAdd(&count[keys.key(i) >> shift & mask], 1u);
  }
  __syncthreads();
  counts[threadIdx.x * tiles + blockIdx.x] = count[threadIdx.x];
}

// One digit's counts become the offsets of its tiles within the digit.
__global__ __launch_bounds__(kThreads) void k_sort_scan(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals,
                                                        uint32_t tiles) {
  __shared__ uint32_t shared[kThreads / kWave + 1];
  uint32_t* mine = counts + (size_t)blockIdx.x * tiles;
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

// A wave's keys follow each other; among the 64 of a round, lanes of equal
// digits find each other by ballots and keep their order.
template <typename K>
__global__ __launch_bounds__(kThreads) void k_sort_scatter(uint32_t* __restrict__ out_keys,
                                                           uint32_t* __restrict__ out_rows, K keys,
                                                           const uint32_t* __restrict__ counts,
                                                           const uint32_t* __restrict__ totals, uint32_t n, int shift,
                                                           uint32_t mask, uint32_t tiles) {
  __shared__ uint32_t count[kSortWaves][kDigits];
  __shared__ uint32_t shared[kThreads / kWave + 1];
  const uint32_t lane = lane_id(), wave = threadIdx.x / kWave;
  for (int w = 0; w < kSortWaves; ++w) count[w][threadIdx.x] = 0;
  uint32_t all;
  const uint32_t start = block_exclusive_u32(totals[threadIdx.x], shared, &all) +
                         counts[threadIdx.x * tiles + blockIdx.x];
  __syncthreads();
  const uint32_t first = blockIdx.x * kSortTile + wave * (kSortTile / kSortWaves) + lane;
  uint32_t key[kSortRounds], rank[kSortRounds];
#pragma unroll
  for (int k = 0; k < kSortRounds; ++k) key[k] = first + k * kWave < n ? keys.key(first + k * kWave) : 0;
#pragma unroll
  for (int k = 0; k < kSortRounds; ++k) {
    const uint32_t digit = key[k] >> shift & mask;
    uint64_t same = __ballot(first + k * kWave < n);
#pragma unroll
    for (int b = 0; b < kDigitBits; ++b) {
      const uint64_t ones = __ballot(digit >> b & 1);
      same &= digit >> b & 1 ? ones : ~ones;
    }
    // Lanes beyond the keys may find no lane; they add and store nothing.
    const int leader = same ? __ffsll((unsigned long long)same) - 1 : (int)lane;
    uint32_t before = 0;
    if (same && leader == (int)lane) before = atomicAdd(&count[wave][digit], (uint32_t)__popcll(same));
    before = __shfl(before, leader, kWave);
    rank[k] = before + (uint32_t)__popcll(same & ((1ull << lane) - 1));
  }
  __syncthreads();
  uint32_t offset = start;
  for (int w = 0; w < kSortWaves; ++w) {
    const uint32_t c = count[w][threadIdx.x];
    count[w][threadIdx.x] = offset;
    offset += c;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSortRounds; ++k) {
    const uint32_t i = first + k * kWave;
    if (i < n) {
      const uint32_t to = count[wave][key[k] >> shift & mask] + rank[k];
      out_keys[to] = key[k];
      out_rows[to] = keys.row(i);
    }
  }
}

// ---- gradient: sums of segments -------------------------------------------

template <typename T>
__global__ __launch_bounds__(kThreads) void k_zero(T* __restrict__ out, int64_t count) {
  constexpr int kSize = Pack<T>::kSize;
  const float zero[kSize] = {};
  for (int64_t at = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kSize; at < count;
       at += (int64_t)gridDim.x * kThreads * kSize)
    store_pack(out, at, count, zero);
}

// A group of kLanes lanes takes `chunk` sorted tokens (its columns by
// blockIdx.y).  A segment that lies inside goes to the table; what belongs to
// a segment of the chunk before goes to heads[chunk], what the next chunks
// continue to tails[chunk] (a chunk inside one segment: heads).
template <typename T, int kLanes>
__global__ __launch_bounds__(kThreads) void k_segment_sums(T* __restrict__ out, float* __restrict__ heads,
                                                           float* __restrict__ tails, const T* __restrict__ grad,
                                                           const uint32_t* __restrict__ keys,
                                                           const uint32_t* __restrict__ rows, uint32_t n,
                                                           uint32_t vocabulary, int64_t dim, int64_t stride,
                                                           float scale, uint32_t chunk, uint32_t chunks) {
  constexpr int kSize = Pack<T>::kSize;
  const int lane = threadIdx.x % kLanes;
  const uint32_t c = blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (c >= chunks) return;
  const int64_t at = ((int64_t)blockIdx.y * kLanes + lane) * kSize;
  const uint32_t begin = c * chunk, end = n - begin < chunk ? n : begin + chunk;
  uint32_t key = keys[begin];
  bool head = begin > 0 && keys[begin - 1] == key;
  float sum[kSize] = {};
  for (uint32_t i = begin; i < end; i += kAhead) {
    float v[kAhead][kSize];
    uint32_t next[kAhead];  // the key after each
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t k = i + j;
      if (k < end) load_pack(grad + (int64_t)rows[k] * stride, at, dim, v[j]);
      next[j] = k + 1 < n ? keys[k + 1] : ~0u;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t k = i + j;
      if (k >= end) break;
#pragma unroll
      for (int e = 0; e < kSize; ++e) sum[e] += v[j][e];
      const bool ends = next[j] != key, last = k + 1 == end;
      if (!ends && !last) continue;
      if (key < vocabulary) {
        if (ends && !head) {
#pragma unroll
          for (int e = 0; e < kSize; ++e) sum[e] *= scale;
          store_pack(out + (int64_t)key * dim, at, dim, sum);
        } else {
          float* to = (head ? heads : tails) + (int64_t)c * dim;
#pragma unroll
          for (int e = 0; e < kSize; ++e)
            if (at + e < dim) to[at + e] = sum[e];
        }
      }
      key = next[j];
      head = false;
#pragma unroll
      for (int e = 0; e < kSize; ++e) sum[e] = 0.0f;
    }
  }
}

// A workgroup for each chunk; where a segment begins in it and goes on, its
// groups share the chunks it runs through.
template <typename T, int kLanes>
__global__ __launch_bounds__(kThreads) void k_segment_join(T* __restrict__ out, const float* __restrict__ heads,
                                                           const float* __restrict__ tails,
                                                           const uint32_t* __restrict__ keys, uint32_t n,
                                                           uint32_t vocabulary, int64_t dim, float scale,
                                                           uint32_t chunk) {
  constexpr int kSize = Pack<T>::kSize;
  constexpr int kGroups = kThreads / kLanes;
  __shared__ float shared[kThreads * kSize];
  const uint32_t c = blockIdx.x;
  const uint32_t begin = c * chunk;
  if (n - begin <= chunk) return;
  const uint32_t end = begin + chunk, key = keys[end];
  // The segment across the chunk's end begins in this chunk, or an earlier one has it.
  if (keys[end - 1] != key || key >= vocabulary) return;
  if (keys[begin] == key && begin > 0 && keys[begin - 1] == key) return;
  uint32_t low = end, high = n;  // the first token beyond the segment
  while (low < high) {
    const uint32_t middle = low + (high - low) / 2;
    if (keys[middle] == key) low = middle + 1;
    else high = middle;
  }
  const uint32_t last = (low - 1) / chunk;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  const int64_t at = ((int64_t)blockIdx.y * kLanes + lane) * kSize;
  float sum[kSize] = {};
  for (uint32_t other = c + 1 + group; other <= last; other += kGroups)
#pragma unroll
    for (int e = 0; e < kSize; ++e)
      if (at + e < dim) sum[e] += heads[(int64_t)other * dim + at + e];
#pragma unroll
  for (int e = 0; e < kSize; ++e) shared[threadIdx.x * kSize + e] = sum[e];
  __syncthreads();
  if (group) return;
#pragma unroll
  for (int e = 0; e < kSize; ++e) sum[e] = at + e < dim ? tails[(int64_t)c * dim + at + e] : 0.0f;
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int e = 0; e < kSize; ++e) sum[e] += shared[(lane + g * kLanes) * kSize + e];
#pragma unroll
  for (int e = 0; e < kSize; ++e) sum[e] *= scale;
  store_pack(out + (int64_t)key * dim, at, dim, sum);
}

// ---- host -------------------------------------------------------------------

// Lanes for a row's columns, a power of two up to a wave.
int row_lanes(int64_t dim, int size) {
  const int64_t packs = (dim + size - 1) / size;
  int lanes = 1;
  while (lanes < kWave && lanes < packs) lanes *= 2;
  return lanes;
}

template <typename F>
void with_lanes(int lanes, F&& fn) {
  switch (lanes) {
    case 1: fn(std::integral_constant<int, 1>()); break;
    case 2: fn(std::integral_constant<int, 2>()); break;
    case 4: fn(std::integral_constant<int, 4>()); break;
    case 8: fn(std::integral_constant<int, 8>()); break;
    case 16: fn(std::integral_constant<int, 16>()); break;
    case 32: fn(std::integral_constant<int, 32>()); break;
    default: fn(std::integral_constant<int, 64>()); break;
  }
}

// Lanes that keep the chip's memory busy: four waves on each SIMD of 256 CUs.
constexpr int64_t kBusyLanes = int64_t(1) << 18;

template <typename T, typename I>
int lookup(T* out, const T* weight, const I* tokens, int64_t rows, int64_t bag, int64_t vocabulary, int64_t dim,
           int64_t stride, float scale, hipStream_t stream) {
  constexpr int kSize = Pack<T>::kSize;
  const int lanes = row_lanes(dim, kSize);
  const int64_t columns = (dim + (int64_t)lanes * kSize - 1) / ((int64_t)lanes * kSize);
  // Few rows: groups share a row's tokens until the chip is busy.
  int split = 1;
  while (split * 2 * lanes <= kThreads && rows * columns * lanes * split < kBusyLanes && (int64_t)split * kAhead < bag)
    split *= 2;
  const int rows_here = kThreads / lanes / split;
  const int64_t wanted = (rows + rows_here - 1) / rows_here;
  const uint32_t grid = (uint32_t)(wanted < (1 << 20) ? wanted : (1 << 20));
  with_lanes(lanes, [&](auto l) {
    constexpr int kLanes = decltype(l)::value;
    if (bag > 1)
      hipLaunchKernelGGL((k_lookup<T, I, kLanes, true>), dim3(grid, (uint32_t)columns), dim3(kThreads), 0, stream, out,
                         weight, tokens, rows, bag, vocabulary, dim, stride, scale, split);
    else
      hipLaunchKernelGGL((k_lookup<T, I, kLanes, false>), dim3(grid, (uint32_t)columns), dim3(kThreads), 0, stream, out,
                         weight, tokens, rows, bag, vocabulary, dim, stride, scale, 1);
  });
  MGB_LAUNCH_CHECK("embedding lookup");
  return 0;
}

// How the gradient of n tokens is laid out in the workspace.
struct GradientPlan {
  uint32_t tiles, chunk, chunks;
  int lanes, passes, bits;
  int64_t columns;
  size_t keys[2], rows[2], counts, totals, heads, tails, bytes;
};

GradientPlan gradient_plan(int64_t n, int64_t vocabulary, int64_t dim, int size) {
  GradientPlan p = {};
  p.tiles = (uint32_t)((n + kSortTile - 1) / kSortTile);
  p.lanes = row_lanes(dim, size);
  p.columns = (dim + (int64_t)p.lanes * size - 1) / ((int64_t)p.lanes * size);
  int bits = 1;
  while (vocabulary >> bits) ++bits;
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  // Sorted tokens of a group: enough groups for the chip, then longer walks,
  // which leave fewer parts to join.
  int64_t chunk = n * p.lanes * p.columns / kBusyLanes;
  chunk = (chunk + kAhead - 1) / kAhead * kAhead;
  p.chunk = (uint32_t)(chunk < kAhead ? kAhead : chunk > 512 ? 512 : chunk);
  p.chunks = (uint32_t)((n + p.chunk - 1) / p.chunk);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t from = at;
    at += (bytes + 255) / 256 * 256;
    return from;
  };
  for (int k = 0; k < 2; ++k) {
    p.keys[k] = take(n * sizeof(uint32_t));
    p.rows[k] = take(n * sizeof(uint32_t));
  }
  p.counts = take((size_t)kDigits * p.tiles * sizeof(uint32_t));
  p.totals = take(kDigits * sizeof(uint32_t));
  p.heads = take((size_t)p.chunks * dim * sizeof(float));
  p.tails = take((size_t)p.chunks * dim * sizeof(float));
  p.bytes = at;
  return p;
}

template <typename K>
void sort_pass(const GradientPlan& p, uint8_t* ws, K keys, uint32_t* out_keys, uint32_t* out_rows, uint32_t n, int pass,
               hipStream_t stream) {
  uint32_t* counts = (uint32_t*)(ws + p.counts);
  uint32_t* totals = (uint32_t*)(ws + p.totals);
  const int shift = pass * p.bits;
  const uint32_t mask = (1u << p.bits) - 1;
  hipLaunchKernelGGL((k_sort_count<K>), dim3(p.tiles), dim3(kThreads), 0, stream, counts, keys, n, shift, mask, p.tiles);
  hipLaunchKernelGGL(k_sort_scan, dim3(kDigits), dim3(kThreads), 0, stream, counts, totals, p.tiles);
  hipLaunchKernelGGL((k_sort_scatter<K>), dim3(p.tiles), dim3(kThreads), 0, stream, out_keys, out_rows, keys, counts,
                     totals, n, shift, mask, p.tiles);
}

template <typename T, typename I>
int lookup_gradient(T* out, const T* grad, const I* tokens, int64_t count, int64_t bag, int64_t vocabulary, int64_t dim,
                    int64_t stride, float scale, uint8_t* ws, hipStream_t stream) {
  constexpr int kSize = Pack<T>::kSize;
  const int64_t packs = (vocabulary * dim + kSize - 1) / kSize, wanted = (packs + kThreads - 1) / kThreads;
  hipLaunchKernelGGL((k_zero<T>), dim3((uint32_t)(wanted < 4096 ? wanted : 4096)), dim3(kThreads), 0, stream, out,
                     vocabulary * dim);
  MGB_LAUNCH_CHECK("embedding gradient: clearing");
  if (count == 0) return 0;
  const GradientPlan p = gradient_plan(count, vocabulary, dim, kSize);
  const uint32_t n = (uint32_t)count;
  uint32_t *keys[2], *rows[2];
  for (int k = 0; k < 2; ++k) {
    keys[k] = (uint32_t*)(ws + p.keys[k]);
    rows[k] = (uint32_t*)(ws + p.rows[k]);
  }
  sort_pass(p, ws, TokenKeys<I>{tokens, (uint32_t)vocabulary, (uint32_t)bag}, keys[0], rows[0], n, 0, stream);
  int now = 0;
  for (int pass = 1; pass < p.passes; ++pass, now ^= 1)
    sort_pass(p, ws, SortedKeys{keys[now], rows[now]}, keys[now ^ 1], rows[now ^ 1], n, pass, stream);
  MGB_LAUNCH_CHECK("embedding gradient: sort");
  float *heads = (float*)(ws + p.heads), *tails = (float*)(ws + p.tails);
  with_lanes(p.lanes, [&](auto l) {
    constexpr int kLanes = decltype(l)::value;
    constexpr uint32_t kGroups = kThreads / kLanes;
    hipLaunchKernelGGL((k_segment_sums<T, kLanes>), dim3((p.chunks + kGroups - 1) / kGroups, (uint32_t)p.columns),
                       dim3(kThreads), 0, stream, out, heads, tails, grad, keys[now], rows[now], n,
                       (uint32_t)vocabulary, dim, stride, scale, p.chunk, p.chunks);
    if (p.chunks > 1)
      hipLaunchKernelGGL((k_segment_join<T, kLanes>), dim3(p.chunks - 1, (uint32_t)p.columns), dim3(kThreads), 0,
                         stream, out, heads, tails, keys[now], n, (uint32_t)vocabulary, dim, scale, p.chunk);
  });
  MGB_LAUNCH_CHECK("embedding gradient: sums");
  return 0;
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

size_t mgb_embedding_gradient_workspace_bytes(int64_t tokens, int64_t vocabulary, int64_t dim, int dtype) {
  if (tokens < 1 || tokens > kMost || vocabulary < 1 || vocabulary > kMost || dim < 1) return 0;
  return gradient_plan(tokens, vocabulary, dim, dtype == MGB_F32 ? 4 : 8).bytes;
}

int mgb_embedding_gradient(void* out, const void* grad, const void* tokens, int64_t rows, int64_t bag,
                           int64_t vocabulary, int64_t dim, int64_t stride, float scale, int dtype, int token_bytes,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (check_sizes(rows, bag, vocabulary, dim, stride)) return -1;
  MGB_REQUIRE(bag == 0 || rows <= kMost / bag, "embedding gradient: tokens must be below 2^31");
  const int64_t count = rows * bag;
  MGB_REQUIRE(out && (count == 0 || (grad && tokens && workspace)), "embedding gradient: null pointer");
  MGB_REQUIRE(workspace_bytes >= mgb_embedding_gradient_workspace_bytes(count, vocabulary, dim, dtype),
              "embedding gradient: workspace too small");
  return with_types(dtype, token_bytes, [&](auto* t, auto* i) {
    using T = std::remove_pointer_t<decltype(t)>;
    using I = std::remove_pointer_t<decltype(i)>;
    return lookup_gradient<T, I>((T*)out, (const T*)grad, (const I*)tokens, count, bag, vocabulary, dim, stride, scale,
                                 (uint8_t*)workspace, (hipStream_t)stream);
  });
}

}  // extern "C"
