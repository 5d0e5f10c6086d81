// The plans of the encoder's products (csrc/feed_forward.hpp), on the host.
//
//   shares   8-bit products of every depth up to 8,192 blocks: the shares of the depth cover it,
//            none is empty and none has more steps than a workgroup holds the scales of.
//            Prints how many plans and how many wrong ones.
//   scales   what a workgroup of an 8-bit product keeps of its operands' scales, for every share of
//            such plans: each row's and column's bytes where its lanes read them.  Behind the last
//            row lies a page that cannot be read.  Prints how many panels and how many wrong bytes.
//   ahead    the panel's steps that are read while others are multiplied: the next one's, and none
//            behind the panel.  Prints how many and how many wrong ones.
//   launches products of up to the most rows that the entries take, of widths of one tile (more do
//            not fit the memory), can be launched: fewer than 2^32 lanes.  Prints how many and how
//            many wrong ones.
#include <sys/mman.h>
#include <unistd.h>

#include <cstdio>
#include <cstring>

#include "feed_forward.hpp"

namespace mgb {
void set_error(std::string) {}
int check(hipError_t, const char*) { return 0; }
}  // namespace mgb

using namespace mgb;
using namespace mgb::block;

namespace {

constexpr int64_t kDepths = 8192;  // a row's blocks

Params product8(int64_t rows, int64_t columns, int64_t blocks, Size* size) {
  Params p = {};
  p.jobs = p.sources = p.pairs = 1;
  p.depth = blocks * 128;
  p.job[0].rows = rows;
  p.job[0].columns = columns;
  Space space = {};
  *size = choose_shares(p, space, false, 128, product::kScaleSteps);
  return p;
}

int shares() {
  const int64_t sizes[][2] = {{33, 1}, {64, 64}, {100, 1024}, {300, 1024}, {512, 8576}, {4096, 1024}, {8192, 8192}, {40000, 70}};
  long plans = 0, wrong = 0;
  for (const auto& s : sizes)
    for (int64_t blocks = 1; blocks <= kDepths; ++blocks, ++plans) {
      Size size;
      const Params p = product8(s[0], s[1], blocks, &size);
      const int64_t before_last = p.splits > 1 ? p.first_steps + int64_t(p.splits - 2) * p.other_steps : 0;
      const int64_t last = blocks - before_last, longest = p.splits > 1 ? p.other_steps : p.first_steps;
      if (p.splits < 1 || p.first_steps < 1 || p.first_steps > product::kScaleSteps || last < 1 || last > longest ||
          longest > product::kScaleSteps)
        ++wrong;
    }
  printf("plans %ld wrong %ld\n", plans, wrong);
  return 0;
}

// `bytes` that end where a page without access begins; what the values are, the place says.
uint8_t* before_a_wall(size_t bytes) {
  const size_t page = sysconf(_SC_PAGESIZE), whole = (bytes + page - 1) / page * page;
  char* const at = (char*)mmap(nullptr, whole + page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
  if (at == MAP_FAILED || mprotect(at + whole, page, PROT_NONE)) return nullptr;
  uint8_t* const begin = (uint8_t*)at + whole - bytes;
  for (size_t k = 0; k < bytes; ++k) begin[k] = (uint8_t)(k * 2654435761u >> 13);
  return begin;
}

template <class S>
long wrong_scales(const Params& p, bool dual, int64_t row0, int64_t column0, uint32_t begin, uint32_t end) {
  using Panel = product::Scales<S>;
  static char panel[Panel::kBytes * product::kScaleSteps];
  const int64_t rows = p.job[0].rows, columns = p.job[0].columns;
  memset(panel, 0, sizeof(panel));
  for (int at = 0; at < (S::kTileM + S::kTileN) * Panel::words(begin, end); ++at)
    Panel::fill_word(panel, at, p, row0, rows, column0, columns, dual, begin, end);
  long wrong = 0;
  for (uint32_t step = begin; step < end; ++step) {
    const uint8_t* const of = (const uint8_t*)panel + (step - begin) * Panel::kBytes;
    for (int half = 0; half < 2; ++half)
      for (int lane = 0; lane < 16; ++lane) {
        for (int wave = 0; wave < S::kWavesM; ++wave)
          for (int tile = 0; tile < S::kTilesM; ++tile) {
            const int64_t row = row0 + half * S::kHalfM + wave * S::kRowsM + tile * 16 + lane;
            const int byte = (wave * 16 + lane) * Panel::kWordsM * 4 + half * S::kTilesM + tile;
            wrong += of[byte] != (row < rows ? p.left_scales[row * p.left_scale_stride + step] : 0x7f);
          }
        for (int wave = 0; wave < S::kWavesN; ++wave)
          for (int tile = 0; tile < S::kTilesN; ++tile) {
            // (a pair's: column 8 a + 4 tile + b of 32 is lane 4 a + b)
            const int in = product::paired<false, S>() ? tile / 2 * 32 + lane / 4 * 8 + tile % 2 * 4 + lane % 4 : tile * 16 + lane;
            const int64_t column = column0 + (dual ? 0 : half * S::kHalfN) + wave * S::kRowsN + in;
            const uint8_t* const scales = p.right_scales[dual ? half : 0];
            const int byte = Panel::kM * 4 + (wave * 16 + lane) * Panel::kWordsN * 4 + half * S::kTilesN + tile;
            wrong += of[byte] != (column < columns ? scales[column * p.right_scale_stride + step] : 0x7f);
          }
      }
  }
  return wrong;
}

template <class S>
long wrong_in_last_tile(const Params& p, bool dual, int64_t blocks) {
  const int64_t row0 = (p.job[0].rows - 1) / S::kTileM * S::kTileM, wide = dual ? S::kHalfN : S::kTileN;
  const int64_t column0 = (p.job[0].columns - 1) / wide * wide;
  long wrong = 0;
  for (uint32_t split = 0; split < p.splits; ++split) {
    const int64_t begin = split ? p.first_steps + int64_t(split - 1) * p.other_steps : 0;
    wrong += wrong_scales<S>(p, dual, row0, column0, begin, std::min(begin + (split ? p.other_steps : p.first_steps), blocks));
  }
  return wrong;
}

int scales() {
  const int64_t sizes[][2] = {{33, 16}, {33, 1024}, {300, 1000}, {512, 200}, {1030, 513}, {4096, 1024}};
  const int64_t depths[] = {1, 2, 3, 4, 5, 7, 8, 15, 16, 18, 31, 34, 43, 59, 63, 64, 65, 67, 71, 97, 128, 157, 300, 1001, 4097};
  long panels = 0, wrong = 0;
  for (const auto& s : sizes)
    for (const int64_t blocks : depths) {
      Size size;
      Params p = product8(s[0], s[1], blocks, &size);
      p.left_scale_stride = p.right_scale_stride = (blocks + 3) / 4 * 4;
      const size_t left = s[0] * p.left_scale_stride, right = s[1] * p.right_scale_stride;
      uint8_t* const walls[3] = {before_a_wall(left), before_a_wall(right), before_a_wall(right)};
      if (!walls[0] || !walls[1] || !walls[2]) return 3;
      p.left_scales = walls[0];
      p.right_scales[0] = walls[1];
      p.right_scales[1] = walls[2];
      wrong += size == kLarge    ? wrong_in_last_tile<product::Large>(p, false, blocks)
               : size == kMedium ? wrong_in_last_tile<product::Medium>(p, false, blocks)
                                 : wrong_in_last_tile<product::Small>(p, false, blocks);
      panels += p.splits;
      if (blocks > product::kScaleSteps) continue;
      p.splits = 1;  // the dual form's, whole
      p.first_steps = (uint32_t)blocks;
      wrong += wrong_in_last_tile<product::Large>(p, true, blocks) + wrong_in_last_tile<product::Medium>(p, true, blocks) +
               wrong_in_last_tile<product::Small>(p, true, blocks);
      panels += 3;
    }
  printf("panels %ld wrong %ld\n", panels, wrong);
  return 0;
}

int ahead() {
  long reads = 0, wrong = 0;
  for (uint32_t steps = 1; steps <= (uint32_t)product::kScaleSteps; ++steps)
    for (uint32_t step = 0; step < steps; ++step, ++reads) {
      const uint32_t next = product::Scales<product::Large>::ahead(step, steps);
      wrong += next >= steps || (step + 1 < steps && next != step + 1);
    }
  printf("reads %ld wrong %ld\n", reads, wrong);
  return 0;
}

int launches() {
  long plans = 0, wrong = 0;
  auto check = [&](const Params& p, Size size, bool dual) {
    int threads = size == kLarge ? product::Large::kThreads : size == kMedium ? product::Medium::kThreads : product::Small::kThreads;
    if (in_parts(p, size)) threads = size == kMedium ? product::PartMedium::kThreads : product::PartSmall::kThreads;
    const uint64_t m = side(size), n = dual ? m / 2 : m;
    const uint64_t tiles = (p.job[0].rows + m - 1) / m * ((p.job[0].columns + n - 1) / n);
    ++plans;
    wrong += p.tiles != tiles || (tiles + 7) / 8 * 8 * p.splits * threads >= uint64_t(1) << 32;
  };
  for (const int64_t rows : {int64_t(1) << 20, int64_t(1) << 28, (int64_t(1) << 29) + 1, (int64_t(1) << 30) - 64, (int64_t(1) << 30) + 1,
                             kMostRows - 1})
    for (const int64_t columns : {1, 8, 32, 33, 64, 65, 128})
      for (const int64_t depth : {8, 64, 512})
        for (const int pairs : {1, 6})
          for (const int sources : {1, 2}) {
            Params p = {};
            p.jobs = 1;
            p.sources = sources;
            p.pairs = pairs;
            p.depth = depth;
            p.job[0].rows = rows;
            p.job[0].columns = columns;
            Size size = choose(p, true);
            check(p, size, true);
            size = choose(p, false);
            check(p, size, false);
            Space space = {};
            for (const bool turned : {false, true}) {
              size = choose_shares(p, space, turned);
              check(p, size, false);
            }
            if (pairs > 1 || depth % 128) continue;
            size = choose(p, true, 128);
            check(p, size, true);
            size = choose_shares(p, space, false, 128, product::kScaleSteps);
            check(p, size, false);
          }
  printf("plans %ld wrong %ld\n", plans, wrong);
  return 0;
}

}  // namespace

int main(int count, char** args) {
  if (count == 2 && !strcmp(args[1], "shares")) return shares();
  if (count == 2 && !strcmp(args[1], "scales")) return scales();
  if (count == 2 && !strcmp(args[1], "ahead")) return ahead();
  if (count == 2 && !strcmp(args[1], "launches")) return launches();
  return 2;
}
