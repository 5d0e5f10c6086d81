// The gated feed-forward block's gradients, from what the forward pass kept:
//   dhidden = dy Wd, dgate = dhidden up act'(gate), dup = dhidden act(gate),
//   dx = dgate Wg + dup Wu, dWg = dgate^T x, dWu = dup^T x, dWd = dy^T hidden.
// dhidden never leaves the registers: the product that has it writes dgate, dup and
// hidden, each rounded to x's type once (to two values of it where results are few).  Its
// end, 214 of its 303 us at 16,384 x 1,024 x 4,096 in bfloat16, is bound by memory.  dx is one product over both matrices'
// rows; the matrices' gradients are one launch, whose operands go along the rows
// and are transposed as they are read from LDS.
#include "feed_forward.hpp"

namespace mgb {
namespace block {
namespace {

// Rows from which on 16-bit matrices are transposed first (gradient(), below).
constexpr int64_t kTurnRows = 4096;

template <typename T, bool kRest>
struct Slope {
  static constexpr bool kDual = false, kBlocks = false;
  static constexpr int kDeep = 4;
  const Params& p;
  int64_t rows;
  __device__ __forceinline__ Slope(const Params& params, const product::Job& job, uint32_t) : p(params), rows(job.rows) {}
  template <int kCount>
  struct Loaded {
    float gate[kCount], up[kCount];
  };
  template <int kCount, bool kWhole, typename L>
  __device__ __forceinline__ void load(L& l, int64_t m, int64_t n) const {
    const float* from = p.kept + (kWhole || m < rows ? m : rows - 1) * 2 * p.true_columns;
    if constexpr (kWhole) {
      __builtin_memcpy(l.gate, from + n, sizeof(l.gate));
      __builtin_memcpy(l.up, from + p.true_columns + n, sizeof(l.up));
    } else {
      load_some<kCount>(from, n, p.true_columns, l.gate);
      load_some<kCount>(from + p.true_columns, n, p.true_columns, l.up);
    }
  }
  template <int kCount, bool kWhole, typename L>
  __device__ __forceinline__ void store(int64_t m, int64_t n, const float* dh, const float*, const L& l) const {
    if (!kWhole && (m >= rows || n >= p.hidden_columns)) return;
    float dgate[kCount], dup[kCount], hidden[kCount];
#pragma unroll
    for (int e = 0; e < kCount; ++e) {
      float slope;
      const float act = activate<sizeof(T) == 4>(l.gate[e], p.activation, &slope);
      const bool there = kWhole || n + e < p.true_columns;  // columns that pad a row are zero whatever dy holds
      hidden[e] = there ? act * l.up[e] : 0.0f;
      dgate[e] = there ? dh[e] * l.up[e] * slope : 0.0f;
      dup[e] = there ? dh[e] * act : 0.0f;
    }
    const int64_t at = m * p.hidden_stride + n;
    store_inner<T, kRest, kCount>(p.dgate, p.gradient_part, p.gradient_rest, at, dgate);
    store_inner<T, kRest, kCount>(p.dgate, p.gradient_part, p.gradient_rest, p.gradient_second + at, dup);
    if (p.hidden) store_inner<T, kRest, kCount>(p.hidden, p.hidden_part, p.hidden_rest, at, hidden);
  }
};

// Gradients of no rows.
__global__ __launch_bounds__(256) void k_clear(uint8_t* a, int64_t a_bytes, uint8_t* b, int64_t b_bytes, uint8_t* c,
                                               int64_t c_bytes) {
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < a_bytes || at < b_bytes || at < c_bytes; at += step) {
    if (at < a_bytes) a[at] = 0;
    if (at < b_bytes) b[at] = 0;
    if (at < c_bytes) c[at] = 0;
  }
}

template <typename T>
int gradient(const MgbFeedForwardGradient& a, Space& space, hipStream_t stream, bool run) {
  using E = typename Kind<T>::E;
  constexpr int kParts = Kind<T>::kParts;
  const bool matrices = a.dgate || a.dup || a.ddown;
  if (a.rows == 0) {
    const int64_t bytes = a.dim * a.hidden * (int64_t)sizeof(T);
    if (run && matrices)
      k_clear<<<1024, 256, 0, stream>>>((uint8_t*)a.dgate, a.dgate ? bytes : 0, (uint8_t*)a.dup, a.dup ? bytes : 0,
                                        (uint8_t*)a.ddown, a.ddown ? bytes : 0);
    MGB_LAUNCH_CHECK("feed forward gradient");
    return 0;
  }
  LayJobs jobs = {};
  // Matrices whose products go along their columns are transposed first where that
  // costs little: binary32 ones, which are laid out anyhow, and others of many rows
  // of x (16,384 x 1,024 x 4,096: two products of 322 and 280 us become 303 and 193,
  // for 18 us of transposing).
  const bool turn_weights = sizeof(T) == 4 || a.rows >= kTurnRows;
  const int64_t dim = padded(a.dim), hidden = padded(a.hidden);
  const bool copy = !lies_well<T>(a.gate, a.hidden, a.dim, a.gate_stride) ||
                    !lies_well<T>(a.up, a.hidden, a.dim, a.up_stride) ||
                    (a.hidden > 1 && a.gate_stride != a.up_stride);
  const Laid grad = lay<T>(space, jobs, a.grad, a.rows, a.dim, a.grad_stride);
  const Laid down = turn_weights ? lay_turned<T>(space, jobs, a.down, a.dim, a.hidden, a.down_stride)
                                 : lay<T>(space, jobs, a.down, a.dim, a.hidden, a.down_stride);
  Laid x = {}, gate = {}, up = {};
  if (a.dgate || a.dup) x = lay<T>(space, jobs, a.x, a.rows, a.dim, a.x_stride);
  if (a.dx && turn_weights) {
    gate = lay_turned<T>(space, jobs, a.gate, a.hidden, a.dim, a.gate_stride);
    up = lay_turned<T>(space, jobs, a.up, a.hidden, a.dim, a.up_stride);
  } else if (a.dx) {
    gate = lay<T>(space, jobs, a.gate, a.hidden, a.dim, a.gate_stride, copy);
    up = lay<T>(space, jobs, a.up, a.hidden, a.dim, a.up_stride, copy);
  }

  const bool halves = sizeof(T) == 2 && std::min(a.rows, a.hidden) * a.dim <= kFewResults;
  Params inner = {};
  inner.jobs = 1;
  inner.sources = 1;
  inner.pairs = Kind<T>::kPairs;
  inner.depth = dim;
  inner.hidden_columns = hidden;
  inner.hidden_stride = inner_stride(hidden);
  inner.hidden_part = a.rows * inner.hidden_stride;
  inner.gradient_second = inner.hidden_part;
  inner.gradient_part = 2 * inner.hidden_part;
  inner.gradient_rest = halves ? inner.gradient_part : 0;
  inner.dgate = space.take(inner.gradient_part * (halves ? 2 : kParts) * 2);
  const Laid dgate = {inner.dgate, inner.hidden_stride * 2, inner.gradient_part * 2};
  const Laid dup = {inner.dgate + inner.gradient_second * 2, inner.hidden_stride * 2, inner.gradient_part * 2};
  Laid middle = {};
  if (a.ddown) {
    inner.hidden_rest = halves ? inner.hidden_part : 0;
    inner.hidden = space.take(inner.hidden_part * (halves ? 2 : kParts) * 2);
    middle = {inner.hidden, inner.hidden_stride * 2, inner.hidden_part * 2};
  }
  inner.kept = const_cast<float*>(a.kept);
  inner.true_columns = a.hidden;
  inner.activation = a.activation;
  inner.job[0].left = operand(grad, a.rows, dim);
  inner.job[0].right = turn_weights ? operand(down, a.hidden, dim) : operand(down, hidden, a.dim);
  inner.job[0].rows = a.rows;
  inner.job[0].columns = a.hidden;  // (tiles end at multiples of 8: they hold the padding too)
  const Size inner_size = choose(inner, false);

  Params input = {};
  Size input_size = kSmall;
  if (a.dx) {
    input.jobs = 1;
    input.sources = halves ? 4 : 2;
    input.pairs = Kind<T>::kPairs;
    input.depth = hidden;
    input.job[0].left = operands(dgate, dup, a.rows, hidden);
    for (int k = 0; k < 2; ++k) input.job[0].left.data[2 + k] += inner.gradient_rest * 2;
    input.job[0].right = turn_weights ? operands(gate, up, a.dim, hidden) : operands(gate, up, dim, a.hidden);
    input.job[0].out = a.dx;
    input.job[0].out_stride = a.dim;
    input.job[0].rows = a.rows;
    input.job[0].columns = a.dim;
    input_size = choose_shares(input, space, !turn_weights);
  }

  Params weights = {};
  Size weights_size = kSmall;
  if (matrices) {
    weights.sources = halves ? 2 : 1;
    weights.pairs = Kind<T>::kPairs;
    weights.depth = a.rows;
    auto add = [&](void* out, const Laid& left, int64_t left_rest, int64_t rows, const Laid& right, int64_t right_rest,
                   int64_t columns) {
      if (!out) return;
      product::Job& job = weights.job[weights.jobs++];
      job.left = operands(left, left, padded(rows), a.rows);
      job.right = operands(right, right, padded(columns), a.rows);
      job.left.data[1] += left_rest * 2;
      job.right.data[1] += right_rest * 2;
      job.out = out;
      job.out_stride = columns;
      job.rows = rows;
      job.columns = columns;
    };
    add(a.dgate, dgate, inner.gradient_rest, a.hidden, x, 0, a.dim);
    add(a.dup, dup, inner.gradient_rest, a.hidden, x, 0, a.dim);
    add(a.ddown, grad, 0, a.dim, middle, inner.hidden_rest, a.hidden);
    weights_size = choose_shares(weights, space, true);
  }
  if (!run) return 0;
  lay_out<T>(jobs, stream);
  auto launch_inner = [&](auto turned) {
    constexpr bool kTurned = decltype(turned)::value;
    if constexpr (sizeof(T) == 2) {
      if (halves) return launch_product<E, T, false, kTurned, Slope<T, true>>(inner, inner_size, stream);
    }
    launch_product<E, T, false, kTurned, Slope<T, false>>(inner, inner_size, stream);
  };
  if (turn_weights) {
    launch_inner(std::bool_constant<false>{});
    if (a.dx) store_product<E, T, T, false, false>(input, input_size, stream);
  } else if constexpr (sizeof(T) == 2) {
    launch_inner(std::bool_constant<true>{});
    if (a.dx) store_product<E, T, T, false, true>(input, input_size, stream);
  }
  if (matrices) store_product<E, T, T, true, true>(weights, weights_size, stream);
  MGB_LAUNCH_CHECK("feed forward gradient");
  return 0;
}

int with_type(const MgbFeedForwardGradient& a, Space& space, hipStream_t stream, bool run) {
  switch (a.dtype) {
    case MGB_F32: return gradient<float>(a, space, stream, run);
    case MGB_F16: return gradient<_Float16>(a, space, stream, run);
    case MGB_BF16: return gradient<__bf16>(a, space, stream, run);
  }
  set_error("feed forward gradient: types must be float32, float16 or bfloat16");
  return -1;
}

int check_sizes(const MgbFeedForwardGradient* a) {
  MGB_REQUIRE(a, "feed forward gradient: null pointer");
  MGB_REQUIRE(a->rows >= 0 && a->rows < kMostRows, "feed forward gradient: rows must be below 2^31 - 2,048");
  MGB_REQUIRE(a->dim >= 1 && a->hidden >= 1 && a->dim <= kMostSide && a->hidden <= kMostSide,
              "feed forward gradient: a matrix' sides must be 1 to 2^20");
  MGB_REQUIRE(a->activation == MGB_SILU || a->activation == MGB_GELU,
              "feed forward gradient: activation must be silu or gelu");
  for (const int64_t stride : {a->grad_stride, a->x_stride, a->gate_stride, a->up_stride, a->down_stride})
    MGB_REQUIRE(stride < (int64_t(1) << 40) && stride > -(int64_t(1) << 40),
                "feed forward gradient: row stride out of range");
  return 0;
}

}  // namespace
}  // namespace block
}  // namespace mgb

using namespace mgb;

extern "C" {

size_t mgb_feed_forward_gradient_workspace_bytes(const MgbFeedForwardGradient* a) {
  if (block::check_sizes(a)) return 0;
  block::Space space = {};
  return block::with_type(*a, space, nullptr, false) ? 0 : space.used;
}

int mgb_feed_forward_gradient(const MgbFeedForwardGradient* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (block::check_sizes(a)) return -1;
  MGB_REQUIRE(a->dtype >= MGB_F32 && a->dtype <= MGB_BF16,
              "feed forward gradient: types must be float32, float16 or bfloat16");
  MGB_REQUIRE(a->rows == 0 || (a->grad && a->x && a->kept && a->gate && a->up && a->down && workspace),
              "feed forward gradient: null pointer");
  MGB_REQUIRE(workspace_bytes >= mgb_feed_forward_gradient_workspace_bytes(a),
              "feed forward gradient: workspace too small");
  MGB_REQUIRE((uintptr_t)workspace % 256 == 0, "feed forward gradient: the workspace must begin at 256 bytes");
  block::Space space = {(char*)workspace, 0};
  return block::with_type(*a, space, (hipStream_t)stream, true);
}

}  // extern "C"
