// Distillation: a row's loss is how far its logits z are from a teacher's largest
// ones, given as values t_j at columns i_j:
//   q = softmax(z / T),  p = softmax over the given j of t / T,
//   loss = T^2 sum_j p_j (log p_j - log q_{i_j}),  dz = grad T (q - p at the i_j).
// An entry whose column lies outside the row is absent; a row without entries has
// loss and gradient 0.  Entries of the same column add up.
//
// Bound by memory: the loss reads z once, with the running largest value and sum of a
// softmax in each lane, 32 bfloat16 values between two changes of it; the gradient
// reads it once and writes dz.  8,192 rows of 32,768 bfloat16: loss 92 us, 5.8 TB/s of
// the logits (a plain read reaches 6.2, one past the caches 7.1); gradient 209 us, 5.1
// TB/s (a large copy 5.0).  Sums are binary32.
#include <algorithm>
#include <type_traits>

#include "encoder_common.hpp"

namespace mgb {
namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.44269504f, kLowest = -3.40282347e38f;
// Logits of this many bytes go past the caches, of whose last level this is the size.
// 8,192 rows of 32,768 in bfloat16 (537 MB): loss 92 us, gradient 209, through the
// caches 98 and 237; a quarter of them 27 and 58, through the caches 28 and 53.
constexpr int64_t kStreamBytes = 256 << 20;
constexpr int64_t kMostClasses = int64_t(1) << 31;

struct Teacher {
  const void* values;
  const void* indices;
  int64_t count, value_stride, index_stride;
  int value_type, index_bytes;

  __device__ __forceinline__ float value(int64_t row, int64_t j) const {
    const int64_t at = row * value_stride + j;
    switch (value_type) {
      case MGB_F32: return ((const float*)values)[at];
      case MGB_F16: return (float)((const _Float16*)values)[at];
      default: return (float)((const __bf16*)values)[at];
    }
  }
  __device__ __forceinline__ int64_t column(int64_t row, int64_t j) const {
    const int64_t at = row * index_stride + j;
    return index_bytes == 4 ? ((const int32_t*)indices)[at] : ((const int64_t*)indices)[at];
  }
};

// The running largest value and the sum of exp((v - largest) / T).
struct Running {
  float largest, sum;
  __device__ __forceinline__ void join(float other_largest, float other_sum, float c) {
    const float most = fmaxf(largest, other_largest);
    sum = sum * __builtin_amdgcn_exp2f((largest - most) * c) + other_sum * __builtin_amdgcn_exp2f((other_largest - most) * c);
    largest = most;
  }
};

// Two of them joined over the lanes of a row; `shared` holds two a wave.
template <int kLanes>
__device__ __forceinline__ void join_lanes(Running& a, Running& b, float c, Running* shared) {
#pragma unroll
  for (int d = (kLanes < kWave ? kLanes : kWave) / 2; d > 0; d /= 2) {
    a.join(__shfl_xor(a.largest, d, kWave), __shfl_xor(a.sum, d, kWave), c);
    b.join(__shfl_xor(b.largest, d, kWave), __shfl_xor(b.sum, d, kWave), c);
  }
  if constexpr (kLanes > kWave) {
    __syncthreads();
    if (threadIdx.x % kWave == 0) {
      shared[threadIdx.x / kWave * 2] = a;
      shared[threadIdx.x / kWave * 2 + 1] = b;
    }
    __syncthreads();
    a = shared[0];
    b = shared[1];
#pragma unroll
    for (int w = 1; w < kLanes / kWave; ++w) {
      a.join(shared[2 * w].largest, shared[2 * w].sum, c);
      b.join(shared[2 * w + 1].largest, shared[2 * w + 1].sum, c);
    }
  }
}

template <int kLanes>
__device__ __forceinline__ float sum_lanes(float v, float* shared) {
  if constexpr (kLanes <= kWave) return group_sum<kLanes>(v);
  else return block_sum<kLanes>(v, shared);
}

// An entry of the teacher's; absent ones have value -inf.
struct Entry {
  int32_t column;
  float value;
};

__device__ __forceinline__ Entry entry_of(const Teacher& teacher, int64_t row, int64_t classes, int64_t j) {
  const int64_t column = teacher.column(row, j);
  const bool there = column >= 0 && column < classes;
  return {there ? (int32_t)column : -1, there ? teacher.value(row, j) : -INFINITY};
}

// A lane's first entry, without a branch on what is fetched.
__device__ __forceinline__ Entry first_entry(const Teacher& teacher, int64_t row, int64_t classes, int lane) {
  if (lane >= teacher.count) return {-1, -INFINITY};
  const int64_t column = teacher.column(row, lane);
  const float value = teacher.value(row, lane);
  const bool there = column >= 0 && column < classes;
  return {there ? (int32_t)column : -1, there ? value : -INFINITY};
}

// A lane's entries (`first` is its first): the largest value and the sum.
template <int kLanes>
__device__ __forceinline__ Running teach(const Teacher& teacher, const Entry& first, int64_t row, int64_t classes, int lane,
                                         float c) {
  Running r = {kLowest, 0.0f};
  for (int64_t j = lane; j < teacher.count; j += kLanes) {
    const float v = j == lane ? first.value : entry_of(teacher, row, classes, j).value;
    if (v != -INFINITY) r.join(v, 1.0f, c);
  }
  return r;
}

// 16 bytes of a row, or from it past the caches.
template <bool kStream, typename T>
__device__ __forceinline__ void load_raw(Raw<T, Pack<T>::kSize>& raw, const T* from) {
  using Loose = __attribute__((ext_vector_type(4), aligned(2))) uint32_t;
  if constexpr (kStream) raw.bits = __builtin_nontemporal_load((const Loose*)from);
  else raw.load(from);
}

template <bool kStream, typename T>
__device__ __forceinline__ void store_raw(const float* v, T* to) {
  using Loose = __attribute__((ext_vector_type(4), aligned(2))) uint32_t;
  T r[Pack<T>::kSize];
#pragma unroll
  for (int e = 0; e < Pack<T>::kSize; ++e) r[e] = (T)v[e];
  Loose bits;
  __builtin_memcpy(&bits, r, sizeof(bits));
  if constexpr (kStream) __builtin_nontemporal_store(bits, (Loose*)to);
  else __builtin_memcpy(to, r, sizeof(r));
}

// The running value and sum of a lane's part of a row, kAhead packs at a time: values
// v count as 2^(c v - base), c = log2(e) / T.
template <bool kStream, typename T, int kLanes>
__device__ __forceinline__ Running sweep(const T* z, int64_t begin, int64_t end, int lane, float c) {
  constexpr int kSize = Pack<T>::kSize, kAhead = 4;
  Running r = {kLowest, 0.0f};
  auto take = [&](const float* v, auto count) {
    constexpr int kCount = decltype(count)::value;
    float most = r.largest;
#pragma unroll
    for (int e = 0; e < kCount; ++e) most = fmaxf(most, v[e]);
    float sum[2] = {r.sum * __builtin_amdgcn_exp2f((r.largest - most) * c), 0.0f};
#pragma unroll
    for (int e = 0; e < kCount; ++e) sum[e % 2] += __builtin_amdgcn_exp2f((v[e] - most) * c);
    r = {most, sum[0] + sum[1]};
  };
  int64_t at = begin + (int64_t)lane * kSize;
  for (; at + (int64_t)(kAhead - 1) * kLanes * kSize + kSize <= end; at += (int64_t)kAhead * kLanes * kSize) {
    Raw<T, kSize> raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) load_raw<kStream>(raw[k], z + at + (int64_t)k * kLanes * kSize);
    float v[kAhead * kSize];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) raw[k].get(v + k * kSize);
    take(v, std::integral_constant<int, kAhead * kSize>{});
  }
  for (; at < end; at += (int64_t)kLanes * kSize) {
    float v[kSize];
    load_pack(z, at, end, v);
#pragma unroll
    for (int e = 0; e < kSize; ++e)
      if (at + e >= end) v[e] = -INFINITY;
    take(v, std::integral_constant<int, kSize>{});
  }
  return r;
}

// log sum exp(z / T), and the row's loss.
template <typename T, int kLanes>
__device__ __forceinline__ void finish_row(float* loss, float* lses, const T* z, const Teacher& teacher,
                                           const Entry& first, Running r, int64_t row, int64_t classes, int lane,
                                           float temperature, float c, Running* shared) {
  const float inverse = 1.0f / temperature;
  const float logit = first.value != -INFINITY ? (float)z[first.column] : 0.0f;
  Running t = teach<kLanes>(teacher, first, row, classes, lane, c);
  join_lanes<kLanes>(r, t, c, shared);
  const float log_sum = logf(r.sum), lse = fmaf(r.largest, inverse, log_sum), log_total = logf(t.sum);
  float sum = 0.0f;
  for (int64_t j = lane; j < teacher.count; j += kLanes) {
    const Entry e = j == lane ? first : entry_of(teacher, row, classes, j);
    if (e.value == -INFINITY) continue;
    const float log_p = (e.value - t.largest) * inverse - log_total, p = expf(log_p);
    const float there = j == lane ? logit : (float)z[e.column];
    // log q from the row's largest logit: lse, rounded, is as far off as the logits are
    // from zero.  (Halves: their difference does not overflow.)
    const float log_q = (0.5f * there - 0.5f * r.largest) * (2.0f * inverse) - log_sum;
    if (p != 0.0f) sum = fmaf(p, log_p - log_q, sum);
  }
  sum = sum_lanes<kLanes>(sum, (float*)shared);
  if (lane == 0) {
    loss[row] = t.sum > 0.0f || t.sum != t.sum ? sum * temperature * temperature : 0.0f;
    lses[row] = lse;
  }
}

// A row by kLanes lanes; with `partial` a part of it, columns blockIdx.y each.
template <bool kStream, typename T, int kLanes>
__global__ __launch_bounds__(kThreads) void k_loss(float* __restrict__ loss, float* __restrict__ lses, Running* __restrict__ partial,
                                                   const T* __restrict__ logits, Teacher teacher, int64_t rows, int64_t classes,
                                                   int64_t stride, int64_t part, float temperature) {
  __shared__ Running shared[2 * kThreads / kWave];
  const int lane = threadIdx.x % kLanes;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  if (row >= rows) return;  // (no barrier follows where a workgroup has several rows)
  const float c = kLog2e / temperature;
  const T* z = logits + row * stride;
  const int64_t begin = (int64_t)blockIdx.y * part, end = begin + part < classes ? begin + part : classes;
  if (partial) {
    Running r = sweep<kStream, T, kLanes>(z, begin, end, lane, c), none = {kLowest, 0.0f};
    join_lanes<kLanes>(r, none, c, shared);
    if (lane == 0) partial[row * gridDim.y + blockIdx.y] = r;
    return;
  }
  const Entry first = first_entry(teacher, row, classes, lane);  // (on its way during the sweep)
  const Running r = sweep<kStream, T, kLanes>(z, begin, end, lane, c);
  finish_row<T, kLanes>(loss, lses, z, teacher, first, r, row, classes, lane, temperature, c, shared);
}

template <typename T>
__global__ __launch_bounds__(kWave) void k_loss_join(float* __restrict__ loss, float* __restrict__ lses,
                                                     const Running* __restrict__ partial, int parts, const T* __restrict__ logits,
                                                     Teacher teacher, int64_t classes, int64_t stride, float temperature) {
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const float c = kLog2e / temperature;
  const T* z = logits + row * stride;
  const Entry first = first_entry(teacher, row, classes, lane);
  Running r = {kLowest, 0.0f};
  for (int k = lane; k < parts; k += kWave) r.join(partial[row * parts + k].largest, partial[row * parts + k].sum, c);
  finish_row<T, kWave>(loss, lses, z, teacher, first, r, row, classes, lane, temperature, c, nullptr);
}

// dz of a part of a row: q everywhere (0 where it is below 2^-126), then the teacher's
// columns once more, by the lane of a column's first entry.  The entries' columns and
// probabilities lie in LDS, and each is compared with all others: 8,192 rows of 32,768 with
// 64 entries 207 us, with 256 292, with 1,024 1,427.
template <bool kStream, typename T, int kLanes>
__global__ __launch_bounds__(kThreads) void k_loss_gradient(T* __restrict__ dz, const float* __restrict__ grad,
                                                            const T* __restrict__ logits, const float* __restrict__ lses,
                                                            Teacher teacher, int64_t rows, int64_t classes, int64_t grad_stride,
                                                            int64_t stride, int64_t part, float temperature) {
  extern __shared__ Entry all_entries[];
  __shared__ Running shared[2 * kThreads / kWave];
  constexpr int kSize = Pack<T>::kSize;
  const int lane = threadIdx.x % kLanes, count = (int)teacher.count;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes;
  const bool there = row < rows;
  if (kLanes > kWave && !there) return;
  Entry* const entries = all_entries + threadIdx.x / kLanes * count;
  const float inverse = 1.0f / temperature;
  const int64_t begin = (int64_t)blockIdx.y * part, end = begin + part < classes ? begin + part : classes;
  float factor = 0.0f, lse = 0.0f;
  bool empty = true;
  const T* z = logits;
  T* out = dz;
  auto slope = [&](float v) { return __builtin_amdgcn_exp2f(fmaf(v, inverse, -lse) * kLog2e); };
  if (there) {
    z = logits + row * stride;
    out = dz + row * classes;
    Running t = teach<kLanes>(teacher, first_entry(teacher, row, classes, lane), row, classes, lane, kLog2e / temperature);
    Running none = {kLowest, 0.0f};
    join_lanes<kLanes>(t, none, kLog2e / temperature, shared);
    const float log_total = logf(t.sum);
    for (int j = lane; j < count; j += kLanes) {
      Entry e = entry_of(teacher, row, classes, j);
      const bool there = e.value != -INFINITY;
      entries[j] = {there ? e.column : -1, there ? expf((e.value - t.largest) * inverse - log_total) : 0.0f};
    }
    empty = t.sum == 0.0f;
    // (Of NaN or an infinity among the teacher's values there are no probabilities: all of the
    // row's gradient is NaN, as its loss is.)
    factor = t.sum == t.sum ? grad[row * grad_stride] * temperature : t.sum;
    lse = lses[row];
    constexpr int kAhead = 4;
    int64_t at = begin + (int64_t)lane * kSize;
    for (; at + (int64_t)(kAhead - 1) * kLanes * kSize + kSize <= end; at += (int64_t)kAhead * kLanes * kSize) {
      Raw<T, kSize> raw[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) load_raw<kStream>(raw[k], z + at + (int64_t)k * kLanes * kSize);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        float v[kSize];
        raw[k].get(v);
#pragma unroll
        for (int e = 0; e < kSize; ++e) v[e] = empty ? 0.0f : factor * slope(v[e]);
        store_raw<kStream>(v, out + at + (int64_t)k * kLanes * kSize);
      }
    }
    for (; at < end; at += (int64_t)kLanes * kSize) {
      float v[kSize];
      load_pack(z, at, end, v);
#pragma unroll
      for (int e = 0; e < kSize; ++e) v[e] = empty ? 0.0f : factor * slope(v[e]);
      store_pack(out, at, end, v);
    }
  }
  __syncthreads();
  if (empty) return;
  for (int j = lane; j < count; j += kLanes) {
    const int32_t column = entries[j].column;
    if (column < begin || column >= end) continue;
    bool first = true;
    float p = 0.0f;
    for (int k = 0; k < count; ++k) {
      const bool same = entries[k].column == column;
      first = first && !(same && k < j);
      p += same ? entries[k].value : 0.0f;
    }
    if (first) out[column] = (T)(factor * (slope((float)z[column]) - p));
  }
}

struct Plan {
  int lanes;       // of a row
  int64_t parts, part;
};

// Rows of up to 2,048 columns, a lane's 4 packs, by a wave, so that no barrier joins
// them; wider ones by a workgroup (8,192 rows of 32,768 by a wave each: 2 % slower);
// where there are too few of those for the chip, in parts of at least 8,192 columns, a
// lane's 4 packs again.
Plan plan(int64_t rows, int64_t classes) {
  Plan p = {classes <= 2048 ? kWave : kThreads, 1, classes};
  if (p.lanes == kThreads && rows < 1024) {
    p.parts = std::max<int64_t>(1, std::min((classes + 8191) / 8192, 1024 / std::max<int64_t>(rows, 1)));
    p.part = ((classes + p.parts - 1) / p.parts + 7) / 8 * 8;
    p.parts = (classes + p.part - 1) / p.part;
  }
  return p;
}

int check_arguments(const MgbDistillation* a) {
  MGB_REQUIRE(a, "distillation: null pointer");
  MGB_REQUIRE(a->rows >= 0 && a->rows < (int64_t(1) << 31), "distillation: rows must be below 2^31");
  MGB_REQUIRE(a->classes >= 1 && a->classes < kMostClasses, "distillation: a row must have 1 to 2^31 - 1 logits");
  MGB_REQUIRE(a->top >= 0 && a->top <= 1024, "distillation: a teacher's row must have at most 1,024 entries");
  MGB_REQUIRE(a->temperature > 0.0f && a->temperature < INFINITY, "distillation: the temperature must be positive");
  MGB_REQUIRE(a->index_bytes == 4 || a->index_bytes == 8, "distillation: indices must be int32 or int64");
  for (const int type : {a->dtype, a->value_dtype})
    MGB_REQUIRE(type >= MGB_F32 && type <= MGB_BF16, "distillation: types must be float32, float16 or bfloat16");
  for (const int64_t stride : {a->stride, a->value_stride, a->index_stride, a->grad_stride})
    MGB_REQUIRE(stride < (int64_t(1) << 40) && stride > -(int64_t(1) << 40), "distillation: row stride out of range");
  return 0;
}

Teacher teacher_of(const MgbDistillation& a) {
  return {a.values, a.indices, a.top, a.value_stride, a.index_stride, a.value_dtype, a.index_bytes};
}

// A launch holds fewer than 2^32 lanes: very many rows take several.
constexpr int64_t kLanesAtOnce = int64_t(1) << 31;

// Rows from `first` on, as many as a launch takes.
MgbDistillation rows_from(const MgbDistillation& a, int64_t first, int64_t most) {
  auto size = [](int type) { return type == MGB_F32 ? 4 : 2; };
  auto at = [](auto* from, int64_t bytes) { return from ? (decltype(from))((const char*)from + bytes) : from; };
  MgbDistillation part = a;
  part.rows = std::min(a.rows - first, most);
  part.loss = at(a.loss, first * 4);
  part.lse = at(a.lse, first * 4);
  part.dlogits = at(a.dlogits, first * a.classes * size(a.dtype));
  part.grad = at(a.grad, first * a.grad_stride * 4);
  part.logits = at(a.logits, first * a.stride * size(a.dtype));
  part.values = at(a.values, first * a.value_stride * size(a.value_dtype));
  part.indices = at(a.indices, first * a.index_stride * a.index_bytes);
  return part;
}

template <typename T>
int loss(const MgbDistillation& a, void* workspace, hipStream_t stream) {
  const Plan p = plan(a.rows, a.classes);
  const bool past_caches = a.rows * a.classes * (int64_t)sizeof(T) >= kStreamBytes;
  Running* partial = p.parts > 1 ? (Running*)workspace : nullptr;  // (of fewer rows than a launch takes)
  for (int64_t done = 0; done < a.rows; done += kLanesAtOnce / p.lanes) {
    const MgbDistillation r = rows_from(a, done, kLanesAtOnce / p.lanes);
    const dim3 grid((uint32_t)((r.rows * p.lanes + kThreads - 1) / kThreads), (uint32_t)p.parts);
    auto launch = [&](auto stream_it, auto lanes) {
      k_loss<decltype(stream_it)::value, T, decltype(lanes)::value><<<grid, kThreads, 0, stream>>>(
          r.loss, r.lse, partial, (const T*)r.logits, teacher_of(r), r.rows, r.classes, r.stride, p.part, r.temperature);
    };
    using Wave = std::integral_constant<int, kWave>;
    using Group = std::integral_constant<int, kThreads>;
    if (p.lanes == kWave) launch(std::false_type{}, Wave{});
    else if (past_caches) launch(std::true_type{}, Group{});
    else launch(std::false_type{}, Group{});
    if (partial)
      k_loss_join<T><<<(uint32_t)r.rows, kWave, 0, stream>>>(r.loss, r.lse, partial, (int)p.parts, (const T*)r.logits,
                                                             teacher_of(r), r.classes, r.stride, r.temperature);
    MGB_LAUNCH_CHECK("distillation loss");
  }
  return 0;
}

template <typename T>
int gradient(const MgbDistillation& a, hipStream_t stream) {
  const Plan p = plan(a.rows, a.classes);
  const bool past_caches = a.rows * a.classes * (int64_t)sizeof(T) >= kStreamBytes;
  const uint32_t lds = (uint32_t)(kThreads / p.lanes * a.top * sizeof(Entry));
  for (int64_t done = 0; done < a.rows; done += kLanesAtOnce / p.lanes) {
    const MgbDistillation r = rows_from(a, done, kLanesAtOnce / p.lanes);
    const dim3 grid((uint32_t)((r.rows * p.lanes + kThreads - 1) / kThreads), (uint32_t)p.parts);
    auto launch = [&](auto stream_it, auto lanes) {
      k_loss_gradient<decltype(stream_it)::value, T, decltype(lanes)::value><<<grid, kThreads, lds, stream>>>(
          (T*)r.dlogits, r.grad, (const T*)r.logits, r.lse, teacher_of(r), r.rows, r.classes, r.grad_stride, r.stride, p.part,
          r.temperature);
    };
    using Wave = std::integral_constant<int, kWave>;
    using Group = std::integral_constant<int, kThreads>;
    if (p.lanes == kWave) launch(std::false_type{}, Wave{});
    else if (past_caches) launch(std::true_type{}, Group{});
    else launch(std::false_type{}, Group{});
    MGB_LAUNCH_CHECK("distillation gradient");
  }
  return 0;
}

}  // namespace
}  // namespace mgb

using namespace mgb;

extern "C" {

size_t mgb_distillation_loss_workspace_bytes(const MgbDistillation* a) {
  if (check_arguments(a) || a->rows == 0) return 0;
  const Plan p = plan(a->rows, a->classes);
  return p.parts > 1 ? (size_t)a->rows * p.parts * sizeof(Running) : 0;
}

int mgb_distillation_loss(const MgbDistillation* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (check_arguments(a)) return -1;
  if (a->rows == 0) return 0;
  const size_t need = mgb_distillation_loss_workspace_bytes(a);
  MGB_REQUIRE(a->loss && a->lse && a->logits && (a->top == 0 || (a->values && a->indices)) && (workspace || need == 0),
              "distillation loss: null pointer");
  MGB_REQUIRE(workspace_bytes >= need, "distillation loss: workspace too small");
  switch (a->dtype) {
    case MGB_F32: return loss<float>(*a, workspace, (hipStream_t)stream);
    case MGB_F16: return loss<_Float16>(*a, workspace, (hipStream_t)stream);
    default: return loss<__bf16>(*a, workspace, (hipStream_t)stream);
  }
}

int mgb_distillation_gradient(const MgbDistillation* a, void* stream) {
  if (check_arguments(a)) return -1;
  if (a->rows == 0) return 0;
  MGB_REQUIRE(a->dlogits && a->grad && a->lse && a->logits && (a->top == 0 || (a->values && a->indices)),
              "distillation gradient: null pointer");
  switch (a->dtype) {
    case MGB_F32: return gradient<float>(*a, (hipStream_t)stream);
    case MGB_F16: return gradient<_Float16>(*a, (hipStream_t)stream);
    default: return gradient<__bf16>(*a, (hipStream_t)stream);
  }
}

}  // extern "C"
