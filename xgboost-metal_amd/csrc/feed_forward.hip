// The encoder's gated feed-forward block, forward:
//   gate = x Wg^T, up = x Wu^T, hidden = act(gate) up, y = hidden Wd^T.
// One product has the tiles of gate and up for the same columns in the same
// workgroup, so that gate and up never leave its registers (but for a gradient,
// which reads them in binary32: rounded to 16 bits they would show in it), the
// second is y's.  hidden is rounded to x's type once, or where results are few to two
// values of it (or stays binary32); sums are binary32.  8,192 x 1,024 x 4,096 in binary16:
// 132 and 68 us, 1.04 and 1.01 PFLOP/s.
#include "few_rows.hpp"

namespace mgb {
namespace block {
namespace {

template <typename T, bool kRest>
struct Gated : product::Plainly {
  static constexpr bool kDual = true;
  const Params& p;
  int64_t rows;
  __device__ __forceinline__ Gated(const Params& params, const product::Job& job, uint32_t) : p(params), rows(job.rows) {}
  template <int kCount, bool kWhole, typename L>
  __device__ __forceinline__ void store(int64_t m, int64_t n, const float* gate, const float* up, const L&) const {
    if (!kWhole && (m >= rows || n >= p.hidden_columns)) return;
    float h[kCount];
#pragma unroll
    for (int e = 0; e < kCount; ++e) {
      const bool there = kWhole || n + e < p.true_columns;  // columns that pad a row are zero whatever x holds
      h[e] = there ? activate<sizeof(T) == 4>(gate[e], p.activation) * up[e] : 0.0f;
    }
    store_inner<T, kRest, kCount>(p.hidden, p.hidden_part, p.hidden_rest, m * p.hidden_stride + n, h);
    if (p.kept) {
      float* to = p.kept + m * 2 * p.true_columns;
      product::store_some<kCount, kWhole>(to, n, p.true_columns, gate);
      product::store_some<kCount, kWhole>(to + p.true_columns, n, p.true_columns, up);
    }
  }
};

template <typename T>
int forward(const MgbFeedForward& a, Space& space, hipStream_t stream, bool run) {
  using E = typename Kind<T>::E;
  const bool halves = sizeof(T) == 2 && a.rows * a.dim <= kFewResults;
  if (a.rows <= kMostFewRows) {
    Few f = {};
    f.x = a.x;
    f.w[0] = a.gate;
    f.w[1] = a.up;
    f.x_stride = a.x_stride;
    f.w_stride[0] = a.gate_stride;
    f.w_stride[1] = a.up_stride;
    f.rows = a.rows;
    f.columns = a.hidden;
    f.depth = a.dim;
    f.out = space.take(a.rows * a.hidden * (halves ? sizeof(float) : sizeof(T)));
    f.kept = a.kept;
    f.activation = a.activation;
    Few g = {};
    g.x = f.out;
    g.w[0] = a.down;
    g.x_stride = a.hidden;
    g.w_stride[0] = a.down_stride;
    g.rows = a.rows;
    g.columns = a.dim;
    g.depth = a.hidden;
    g.out = a.y;
    if (run) {
      if (halves) {
        few_rows<Plain<T>, Plain<T>, float, true>(f, stream);
        few_rows<std::conditional_t<sizeof(T) == 2, Halves<T>, Plain<T>>, Plain<T>, T, false>(g, stream);
      } else {
        few_rows<Plain<T>, Plain<T>, T, true>(f, stream);
        few_rows<Plain<T>, Plain<T>, T, false>(g, stream);
      }
      MGB_LAUNCH_CHECK("feed forward");
    }
    return 0;
  }
  LayJobs jobs = {};
  const bool copy = !lies_well<T>(a.gate, a.hidden, a.dim, a.gate_stride) ||
                    !lies_well<T>(a.up, a.hidden, a.dim, a.up_stride) ||
                    (a.hidden > 1 && a.gate_stride != a.up_stride);
  const Laid x = lay<T>(space, jobs, a.x, a.rows, a.dim, a.x_stride);
  const Laid gate = lay<T>(space, jobs, a.gate, a.hidden, a.dim, a.gate_stride, copy);
  const Laid up = lay<T>(space, jobs, a.up, a.hidden, a.dim, a.up_stride, copy);
  const Laid down = lay<T>(space, jobs, a.down, a.dim, a.hidden, a.down_stride);
  const int64_t dim = padded(a.dim), hidden = padded(a.hidden);

  Params inner = {};
  inner.jobs = 1;
  inner.sources = 1;
  inner.pairs = Kind<T>::kPairs;
  inner.depth = dim;
  inner.hidden_columns = hidden;
  inner.hidden_stride = inner_stride(hidden);
  inner.hidden_part = a.rows * inner.hidden_stride;
  inner.hidden_rest = halves ? inner.hidden_part : 0;
  inner.hidden = space.take(inner.hidden_part * (halves ? 2 : Kind<T>::kParts) * 2);
  inner.kept = a.kept;
  inner.true_columns = a.hidden;
  inner.activation = a.activation;
  inner.job[0].left = operand(x, a.rows, dim);
  inner.job[0].right = operands(gate, up, a.hidden, dim);
  inner.job[0].rows = a.rows;
  inner.job[0].columns = a.hidden;  // (tiles end at multiples of 8: they hold the padding too)
  const Size inner_size = choose(inner, true);

  Params outer = {};
  outer.jobs = 1;
  outer.sources = halves ? 2 : 1;
  outer.pairs = Kind<T>::kPairs;
  outer.depth = hidden;
  const Laid middle = {inner.hidden, inner.hidden_stride * 2, inner.hidden_part * 2};
  outer.job[0].left = operands(middle, {inner.hidden + inner.hidden_rest * 2, middle.stride, 0}, a.rows, hidden);
  outer.job[0].left.part = middle.part;
  outer.job[0].right = operands(down, down, a.dim, hidden);
  outer.job[0].out = a.y;
  outer.job[0].out_stride = a.dim;
  outer.job[0].rows = a.rows;
  outer.job[0].columns = a.dim;
  const Size outer_size = choose_shares(outer, space, false);
  if (!run) return 0;
  lay_out<T>(jobs, stream);
  if constexpr (sizeof(T) == 2) {
    if (halves) launch_product<E, T, false, false, Gated<T, true>>(inner, inner_size, stream);
    else launch_product<E, T, false, false, Gated<T, false>>(inner, inner_size, stream);
  } else {
    launch_product<E, T, false, false, Gated<T, false>>(inner, inner_size, stream);
  }
  store_product<E, T, T, false, false>(outer, outer_size, stream);
  MGB_LAUNCH_CHECK("feed forward");
  return 0;
}

int with_type(const MgbFeedForward& a, Space& space, hipStream_t stream, bool run) {
  switch (a.dtype) {
    case MGB_F32: return forward<float>(a, space, stream, run);
    case MGB_F16: return forward<_Float16>(a, space, stream, run);
    case MGB_BF16: return forward<__bf16>(a, space, stream, run);
  }
  set_error("feed forward: types must be float32, float16 or bfloat16");
  return -1;
}

int check_sizes(const MgbFeedForward* a) {
  MGB_REQUIRE(a, "feed forward: null pointer");
  MGB_REQUIRE(a->rows >= 0 && a->rows < kMostRows, "feed forward: rows must be below 2^31 - 2,048");
  MGB_REQUIRE(a->dim >= 1 && a->hidden >= 1 && a->dim <= kMostSide && a->hidden <= kMostSide,
              "feed forward: a matrix' sides must be 1 to 2^20");
  MGB_REQUIRE(a->activation == MGB_SILU || a->activation == MGB_GELU, "feed forward: activation must be silu or gelu");
  for (const int64_t stride : {a->x_stride, a->gate_stride, a->up_stride, a->down_stride})
    MGB_REQUIRE(stride < (int64_t(1) << 40) && stride > -(int64_t(1) << 40), "feed forward: row stride out of range");
  return 0;
}

}  // namespace
}  // namespace block
}  // namespace mgb

using namespace mgb;

extern "C" {

size_t mgb_feed_forward_workspace_bytes(const MgbFeedForward* a) {
  if (block::check_sizes(a) || a->rows == 0) return 0;
  block::Space space = {};
  return block::with_type(*a, space, nullptr, false) ? 0 : space.used;
}

int mgb_feed_forward(const MgbFeedForward* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (block::check_sizes(a)) return -1;
  MGB_REQUIRE(a->dtype >= MGB_F32 && a->dtype <= MGB_BF16, "feed forward: types must be float32, float16 or bfloat16");
  if (a->rows == 0) return 0;
  MGB_REQUIRE(a->y && a->x && a->gate && a->up && a->down && workspace, "feed forward: null pointer");
  MGB_REQUIRE(workspace_bytes >= mgb_feed_forward_workspace_bytes(a), "feed forward: workspace too small");
  MGB_REQUIRE((uintptr_t)workspace % 256 == 0, "feed forward: the workspace must begin at 256 bytes");
  block::Space space = {(char*)workspace, 0};
  return block::with_type(*a, space, (hipStream_t)stream, true);
}

}  // extern "C"
