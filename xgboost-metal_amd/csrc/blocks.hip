// Products in 8 bits with a scale for each block of 128 values, and the encoder's
// block served that way.
//
// A row's values are kept as e4m3 (4 bits of exponent, 3 of mantissa, up to 448), each
// 128 of them times the smallest power of two that takes the largest to at most 448.
// A power of two scales without rounding, is a byte, and is what the matrix
// instruction applies by itself: a step of a product is one block, and its sums need
// no other arithmetic.  Padding to whole blocks is zeros.
//
// The 8-bit instructions add a few products at a time with about 16 bits (1.5e-5 of
// the norm for normal values, whatever the depth), which 16-bit results do not show.
// Binary32 results, and the hidden values of a block in binary32 and binary16, or if
// they are few (they are rounded to e4m3 next: what crosses a border there shows), come
// of the bfloat16 instructions, which take e4m3 values with their scales exactly.
#include "few_rows.hpp"

namespace mgb {
namespace block {
namespace {

// Hidden values from which on bfloat16 rows go by the 8-bit instructions.  64 rows of
// 1,024 x 4,096: 35 us exactly, 23 by them, which is what the 16-bit block takes; 300 of
// 512 x 1,024: 23 and 19.
constexpr int64_t kManyHidden = int64_t(1) << 21;

constexpr int kBlock = 128, kQuantThreads = 256, kQuantLanes = kBlock / 8;

__device__ __forceinline__ float group_max16(float v) {
  v = fmaxf(v, lane_move<0xb1>(v));
  v = fmaxf(v, lane_move<0x4e>(v));
  v = fmaxf(v, lane_move<0x141>(v));
  return fmaxf(v, lane_move<0x140>(v));
}

// 16 lanes a block of 128, 8 values a lane.
template <typename T>
__global__ __launch_bounds__(kQuantThreads) void k_quantize(uint8_t* __restrict__ values, uint8_t* __restrict__ scales,
                                                            const T* __restrict__ x, int64_t rows, int64_t dim,
                                                            int64_t stride, int64_t blocks, int64_t value_stride,
                                                            int64_t scale_stride) {
  const int64_t all = rows * blocks, step = (int64_t)gridDim.x * (kQuantThreads / kQuantLanes);
  const int64_t step_rows = step / blocks, step_blocks = step % blocks;
  const int lane = threadIdx.x % kQuantLanes;
  int64_t at = (int64_t)blockIdx.x * (kQuantThreads / kQuantLanes) + threadIdx.x / kQuantLanes;
  int64_t row = at / blocks, block = at % blocks;
  for (; at < all; at += step) {
    float v[8];
    load_some<8>(x + row * stride, block * kBlock + lane * 8, dim, v);
    float largest = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.0f);
    const uint32_t scale = scale_of(group_max16(largest));
    const uint2 word = round_eight(v, __uint_as_float((254u - scale) << 23));
    __builtin_memcpy(__builtin_assume_aligned(values + row * value_stride + block * kBlock + lane * 8, 8), &word, 8);
    if (lane == 0) scales[row * scale_stride + block] = (uint8_t)scale;
    row += step_rows;
    block += step_blocks;
    if (block >= blocks) {
      block -= blocks;
      ++row;
    }
  }
}

template <typename T>
void quantize(uint8_t* values, uint8_t* scales, const T* x, int64_t rows, int64_t dim, int64_t stride, int64_t value_stride,
              int64_t scale_stride, hipStream_t stream) {
  const int64_t blocks = (dim + kBlock - 1) / kBlock, each = kQuantThreads / kQuantLanes;
  const int64_t groups = std::min<int64_t>((rows * blocks + each - 1) / each, 4096);
  k_quantize<T><<<(uint32_t)groups, kQuantThreads, 0, stream>>>(values, scales, x, rows, dim, stride, blocks, value_stride,
                                                                 scale_stride);
}

// What blocks stand for, as bfloat16, which has their bits and exponents; matrices
// blockIdx.y.
struct Widen {
  __bf16* to[3];
  MgbBlocks m[3];
  int count;
};

__global__ __launch_bounds__(kQuantThreads) void k_widen(Widen w) {
  const MgbBlocks& m = w.m[blockIdx.y];
  const int64_t all = m.rows * m.blocks, step = (int64_t)gridDim.x * (kQuantThreads / kQuantLanes);
  const int lane = threadIdx.x % kQuantLanes;
  for (int64_t at = (int64_t)blockIdx.x * (kQuantThreads / kQuantLanes) + threadIdx.x / kQuantLanes; at < all; at += step) {
    const int64_t row = at / m.blocks, block = at % m.blocks;
    uint2 bytes;
    __builtin_memcpy(&bytes, (const uint8_t*)m.values + row * m.stride + block * kBlock + lane * 8, 8);
    const product::bf16x8 v = widen_eight(bytes, ((const uint8_t*)m.scales)[row * m.scale_stride + block]);
    __builtin_memcpy(w.to[blockIdx.y] + (row * m.blocks + block) * kBlock + lane * 8, &v, sizeof(v));
  }
}

Laid widened(Space& space, Widen& w, const MgbBlocks& m) {
  const int64_t width = m.blocks * kBlock * 2;
  char* to = space.take(m.rows * width);
  w.to[w.count] = (__bf16*)to;
  w.m[w.count++] = m;
  return {to, width, 0};
}

void widen(const Widen& w, hipStream_t stream) {
  const int64_t each = kQuantThreads / kQuantLanes;
  int64_t most = 0;
  for (int k = 0; k < w.count; ++k) most = std::max(most, w.m[k].rows * w.m[k].blocks);
  k_widen<<<dim3((uint32_t)std::min<int64_t>((most + each - 1) / each, 4096), w.count), kQuantThreads, 0, stream>>>(w);
}

product::Operand operand8(const MgbBlocks& m) {
  return {{(const char*)m.values, nullptr}, {m.stride, m.stride}, 0, m.rows, m.blocks * kBlock};
}

// out = x weight^T.  The depth's steps are blocks, of which a workgroup holds the
// scales of kScaleSteps.
template <typename T>
int multiply(T* out, const MgbBlocks& x, const MgbBlocks& weight, Space& space, hipStream_t stream, bool run) {
  if (x.rows <= kMostFewRows) {
    Few f = {};
    f.x = x.values;
    f.w[0] = weight.values;
    f.x_scales = (const uint8_t*)x.scales;
    f.w_scales[0] = (const uint8_t*)weight.scales;
    f.x_stride = x.stride;
    f.w_stride[0] = weight.stride;
    f.x_scale_stride = x.scale_stride;
    f.w_scale_stride = weight.scale_stride;
    f.rows = x.rows;
    f.columns = weight.rows;
    f.depth = x.blocks * kBlock;
    f.out = out;
    if (run) few_rows<InBlocks, InBlocks, T, false>(f, stream);
    return 0;
  }
  Params p = {};
  p.jobs = 1;
  p.sources = 1;
  p.pairs = 1;
  p.depth = x.blocks * kBlock;
  p.job[0].out = out;
  p.job[0].out_stride = weight.rows;
  p.job[0].rows = x.rows;
  p.job[0].columns = weight.rows;
  if constexpr (sizeof(T) == 4) {
    Widen w = {};
    const Laid left = widened(space, w, x), right = widened(space, w, weight);
    if (run) widen(w, stream);
    p.job[0].left = operand(left, x.rows, p.depth);
    p.job[0].right = operand(right, weight.rows, p.depth);
    const Size size = choose_shares(p, space, false);
    if (run) store_product<__bf16, __bf16, T, false, false>(p, size, stream);
  } else {
    p.job[0].left = operand8(x);
    p.job[0].right = operand8(weight);
    p.left_scales = (const uint8_t*)x.scales;
    p.right_scales[0] = (const uint8_t*)weight.scales;
    p.left_scale_stride = x.scale_stride;
    p.right_scale_stride = weight.scale_stride;
    const Size size = choose_shares(p, space, false, kBlock, product::kScaleSteps);
    if (run) store_product<product::E4m3, uint8_t, T, false, false>(p, size, stream);
  }
  return 0;
}

struct GatedFloat : product::Plainly {
  static constexpr bool kDual = true;
  const Params& p;
  int64_t rows;
  __device__ __forceinline__ GatedFloat(const Params& params, const product::Job& job, uint32_t) : p(params), rows(job.rows) {}
  template <int kCount, bool kWhole, typename L>
  __device__ __forceinline__ void store(int64_t m, int64_t n, const float* gate, const float* up, const L&) const {
    if (!kWhole && m >= rows) return;
    float h[kCount];
#pragma unroll
    for (int e = 0; e < kCount; ++e) h[e] = activate<true>(gate[e], p.activation) * up[e];
    product::store_some<kCount, kWhole>((float*)p.hidden + m * p.hidden_stride, n, p.true_columns, h);
  }
};

// The same rounded to blocks in the workgroup that has them: large tiles, whose 128
// columns of both products are a block.
struct GatedBlocks : product::Plainly {
  static constexpr bool kDual = true, kBlocks = true;
  const Params& p;
  __device__ __forceinline__ GatedBlocks(const Params& params, const product::Job&, uint32_t) : p(params) {}
  __device__ __forceinline__ float value(float gate, float up) const { return activate<true>(gate, p.activation) * up; }
  __device__ __forceinline__ void store(int64_t m, int64_t n, uint32_t block, const float* v, float top, bool first) const {
    const uint32_t scale = scale_of(top);
    const uint2 bytes = round_eight(v, __uint_as_float((254u - scale) << 23));
    __builtin_memcpy(__builtin_assume_aligned(p.hidden + m * p.hidden_stride + n, 8), &bytes, 8);
    if (first) p.dgate[m * p.gradient_part + block] = (char)scale;
  }
};

template <class E, class Finish>
void launch_small(const Params& p, Size size, hipStream_t stream) {
  const uint32_t groups = (p.tiles + 7) / 8 * 8 * p.splits;
  if (size == kMedium) product::k_product<E, false, false, product::Medium, Finish><<<groups, product::Medium::kThreads, 0, stream>>>(p);
  else product::k_product<E, false, false, product::Small, Finish><<<groups, product::Small::kThreads, 0, stream>>>(p);
}

template <class E>
void launch_blocks(const Params& p, hipStream_t stream) {
  product::k_product<E, false, false, product::Large, GatedBlocks>
      <<<(p.tiles + 7) / 8 * 8 * p.splits, product::Large::kThreads, 0, stream>>>(p);
}

template <typename T>
int serve(const MgbBlockFeedForward& a, Space& space, hipStream_t stream, bool run) {
  if (a.rows <= kMostFewRows) {
    Few f = {};
    f.x = a.x;
    f.w[0] = a.gate.values;
    f.w[1] = a.up.values;
    f.w_scales[0] = (const uint8_t*)a.gate.scales;
    f.w_scales[1] = (const uint8_t*)a.up.scales;
    f.x_stride = a.x_stride;
    f.w_stride[0] = a.gate.stride;
    f.w_stride[1] = a.up.stride;
    f.w_scale_stride = a.gate.scale_stride;
    f.rows = a.rows;
    f.columns = a.hidden;
    f.depth = a.dim;
    f.out = space.take(a.rows * a.hidden * sizeof(float));
    f.activation = a.activation;
    if (run) few_rows<Rounded<T>, InBlocks, float, true>(f, stream);
    Few g = {};
    g.x = f.out;
    g.w[0] = a.down.values;
    g.w_scales[0] = (const uint8_t*)a.down.scales;
    g.x_stride = a.hidden;
    g.w_stride[0] = a.down.stride;
    g.w_scale_stride = a.down.scale_stride;
    g.rows = a.rows;
    g.columns = a.dim;
    g.depth = a.hidden;
    g.out = a.y;
    if (run) few_rows<Rounded<float>, InBlocks, T, false>(g, stream);
    return 0;
  }
  const int64_t dim = a.gate.blocks * kBlock, hidden = a.down.blocks * kBlock;
  const int64_t x_scales = (a.gate.blocks + 3) / 4 * 4, hidden_scales = (a.down.blocks + 3) / 4 * 4;
  MgbBlocks x = {space.take(a.rows * dim), space.take(a.rows * x_scales), a.rows, a.gate.blocks, dim, x_scales};
  if (run) quantize<T>((uint8_t*)x.values, (uint8_t*)x.scales, (const T*)a.x, a.rows, a.dim, a.x_stride, dim, x_scales, stream);
  Params p = {};
  p.jobs = 1;
  p.sources = 1;
  p.pairs = 1;
  p.depth = dim;
  p.true_columns = a.hidden;
  MgbBlocks h = {space.take(a.rows * hidden), space.take(a.rows * hidden_scales), a.rows, a.down.blocks, hidden, hidden_scales};
  p.activation = a.activation;
  p.job[0].rows = a.rows;
  p.job[0].columns = a.hidden;
  // Bfloat16 rows go by the 8-bit instructions, if their scales are no more than a
  // workgroup holds, the others, exactly, by bfloat16's.  Of the former's hidden values
  // one in a thousand falls on the other side of a border of e4m3's and is a sixteenth
  // off: of many that adds a third to the result's rounding, of few up to as much again.
  const bool in_eight = std::is_same_v<T, __bf16> && a.gate.blocks <= product::kScaleSteps &&
                        a.rows * a.hidden >= kManyHidden;
  const Size size = choose(p, true, in_eight ? kBlock : 64);
  const bool rounds = size == kLarge;
  if (rounds) {
    p.hidden = (char*)h.values;
    p.hidden_stride = hidden;
    p.dgate = (char*)h.scales;
    p.gradient_part = hidden_scales;
  } else {
    p.hidden_stride = a.hidden;
    p.hidden = space.take(a.rows * a.hidden * sizeof(float));
  }
  if (in_eight) {
    p.job[0].left = operand8(x);
    p.job[0].right = {{(const char*)a.gate.values, (const char*)a.up.values}, {a.gate.stride, a.up.stride}, 0, a.hidden, dim};
    p.left_scales = (const uint8_t*)x.scales;
    p.right_scales[0] = (const uint8_t*)a.gate.scales;
    p.right_scales[1] = (const uint8_t*)a.up.scales;
    p.left_scale_stride = x.scale_stride;
    p.right_scale_stride = a.gate.scale_stride;
    if (run && rounds) launch_blocks<product::E4m3>(p, stream);
    else if (run) launch_small<product::E4m3, GatedFloat>(p, size, stream);
  } else {
    Widen w = {};
    const Laid left = widened(space, w, x), gate = widened(space, w, a.gate), up = widened(space, w, a.up);
    if (run) widen(w, stream);
    p.job[0].left = operand(left, a.rows, dim);
    p.job[0].right = operands(gate, up, a.hidden, dim);
    if (run && rounds) launch_blocks<__bf16>(p, stream);
    else if (run) launch_small<__bf16, GatedFloat>(p, size, stream);
  }
  if (run && !rounds)
    quantize<float>((uint8_t*)h.values, (uint8_t*)h.scales, (const float*)p.hidden, a.rows, a.hidden, a.hidden, hidden,
                    hidden_scales, stream);
  return multiply<T>((T*)a.y, h, a.down, space, stream, run);
}

template <class Call>
int with_type(int dtype, const Call& call) {
  switch (dtype) {
    case MGB_F32: return call((float*)nullptr);
    case MGB_F16: return call((_Float16*)nullptr);
    case MGB_BF16: return call((__bf16*)nullptr);
  }
  set_error("blocks: types must be float32, float16 or bfloat16");
  return -1;
}

int check_blocks(const MgbBlocks& m) {
  MGB_REQUIRE(m.rows >= 0 && m.rows < kMostRows, "blocks: rows must be below 2^31 - 2,048");
  MGB_REQUIRE(m.blocks >= 1 && m.blocks <= kMostSide / kBlock, "blocks: a row must have 1 to 8,192 blocks");
  MGB_REQUIRE(m.stride >= m.blocks * kBlock && m.stride <= kMostSide && m.stride % 16 == 0,
              "blocks: rows of values must be 16-byte multiples apart, at most 2^20");
  MGB_REQUIRE(m.scale_stride >= (m.blocks + 3) / 4 * 4 && m.scale_stride % 4 == 0,
              "blocks: rows of scales must be whole words");
  MGB_REQUIRE((uintptr_t)m.values % 16 == 0 && (uintptr_t)m.scales % 4 == 0, "blocks: values must begin at 16 bytes, scales at 4");
  return 0;
}

int check_matmul(const MgbBlockMatmul* a) {
  MGB_REQUIRE(a, "block matmul: null pointer");
  if (check_blocks(a->x) || check_blocks(a->weight)) return -1;
  MGB_REQUIRE(a->x.blocks == a->weight.blocks, "block matmul: both must have the same blocks a row");
  MGB_REQUIRE(a->weight.rows <= kMostSide, "block matmul: a weight must have at most 2^20 rows");
  MGB_REQUIRE(a->dtype >= MGB_F32 && a->dtype <= MGB_BF16, "block matmul: types must be float32, float16 or bfloat16");
  return 0;
}

int check_serve(const MgbBlockFeedForward* a) {
  MGB_REQUIRE(a, "block feed forward: null pointer");
  if (check_blocks(a->gate) || check_blocks(a->up) || check_blocks(a->down)) return -1;
  MGB_REQUIRE(a->rows >= 0 && a->rows < kMostRows, "block feed forward: rows must be below 2^31 - 2,048");
  MGB_REQUIRE(a->dim >= 1 && a->hidden >= 1 && a->dim <= kMostSide && a->hidden <= kMostSide,
              "block feed forward: a matrix' sides must be 1 to 2^20");
  MGB_REQUIRE(a->gate.rows == a->hidden && a->up.rows == a->hidden && a->down.rows == a->dim &&
                  a->gate.blocks == (a->dim + kBlock - 1) / kBlock && a->up.blocks == a->gate.blocks &&
                  a->down.blocks == (a->hidden + kBlock - 1) / kBlock,
              "block feed forward: the matrices' sizes do not fit");
  MGB_REQUIRE(a->gate.stride == a->up.stride && a->gate.scale_stride == a->up.scale_stride,
              "block feed forward: gate and up must lie alike");
  MGB_REQUIRE(a->activation == MGB_SILU || a->activation == MGB_GELU, "block feed forward: activation must be silu or gelu");
  MGB_REQUIRE(a->dtype >= MGB_F32 && a->dtype <= MGB_BF16, "block feed forward: types must be float32, float16 or bfloat16");
  MGB_REQUIRE(a->x_stride < (int64_t(1) << 40) && a->x_stride > -(int64_t(1) << 40), "block feed forward: row stride out of range");
  return 0;
}

}  // namespace
}  // namespace block
}  // namespace mgb

using namespace mgb;

extern "C" {

int mgb_quantize_blocks(const MgbBlocks* out, const void* x, int64_t dim, int64_t x_stride, int dtype, void* stream) {
  MGB_REQUIRE(out, "quantize blocks: null pointer");
  if (block::check_blocks(*out)) return -1;
  MGB_REQUIRE(dim >= 1 && out->blocks == (dim + block::kBlock - 1) / block::kBlock,
              "quantize blocks: a row's blocks must hold its values");
  MGB_REQUIRE(x_stride < (int64_t(1) << 40) && x_stride > -(int64_t(1) << 40), "quantize blocks: row stride out of range");
  MGB_REQUIRE(dtype >= MGB_F32 && dtype <= MGB_BF16, "quantize blocks: types must be float32, float16 or bfloat16");
  if (out->rows == 0) return 0;
  MGB_REQUIRE(out->values && out->scales && x, "quantize blocks: null pointer");
  return block::with_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    block::quantize<T>((uint8_t*)out->values, (uint8_t*)out->scales, (const T*)x, out->rows, dim, x_stride, out->stride,
                       out->scale_stride, (hipStream_t)stream);
    MGB_LAUNCH_CHECK("quantize blocks");
    return 0;
  });
}

size_t mgb_block_matmul_workspace_bytes(const MgbBlockMatmul* a) {
  if (block::check_matmul(a) || a->x.rows == 0 || a->weight.rows == 0) return 0;
  block::Space space = {};
  block::with_type(a->dtype, [&](auto* t) { return block::multiply(t, a->x, a->weight, space, nullptr, false); });
  return space.used;
}

int mgb_block_matmul(const MgbBlockMatmul* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (block::check_matmul(a)) return -1;
  if (a->x.rows == 0 || a->weight.rows == 0) return 0;
  const size_t need = mgb_block_matmul_workspace_bytes(a);
  MGB_REQUIRE(a->out && a->x.values && a->x.scales && a->weight.values && a->weight.scales && (workspace || need == 0),
              "block matmul: null pointer");
  MGB_REQUIRE(workspace_bytes >= need, "block matmul: workspace too small");
  MGB_REQUIRE((uintptr_t)workspace % 256 == 0, "block matmul: the workspace must begin at 256 bytes");
  block::Space space = {(char*)workspace, 0};
  return block::with_type(a->dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (block::multiply((T*)a->out, a->x, a->weight, space, (hipStream_t)stream, true)) return -1;
    MGB_LAUNCH_CHECK("block matmul");
    return 0;
  });
}

size_t mgb_block_feed_forward_workspace_bytes(const MgbBlockFeedForward* a) {
  if (block::check_serve(a) || a->rows == 0) return 0;
  block::Space space = {};
  block::with_type(a->dtype, [&](auto* t) {
    return block::serve<std::remove_pointer_t<decltype(t)>>(*a, space, nullptr, false);
  });
  return space.used;
}

int mgb_block_feed_forward(const MgbBlockFeedForward* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (block::check_serve(a)) return -1;
  if (a->rows == 0) return 0;
  MGB_REQUIRE(a->y && a->x && a->gate.values && a->gate.scales && a->up.values && a->up.scales && a->down.values &&
                  a->down.scales && workspace,
              "block feed forward: null pointer");
  MGB_REQUIRE(workspace_bytes >= mgb_block_feed_forward_workspace_bytes(a), "block feed forward: workspace too small");
  MGB_REQUIRE((uintptr_t)workspace % 256 == 0, "block feed forward: the workspace must begin at 256 bytes");
  block::Space space = {(char*)workspace, 0};
  return block::with_type(a->dtype, [&](auto* t) {
    if (block::serve<std::remove_pointer_t<decltype(t)>>(*a, space, (hipStream_t)stream, true)) return -1;
    MGB_LAUNCH_CHECK("block feed forward");
    return 0;
  });
}

}  // extern "C"
