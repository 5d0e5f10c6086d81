// The plans of the encoder's products (csrc/feed_forward.hpp), on the host.
//
//   shares   8-bit products of every depth up to 8,192 blocks: the shares of the depth cover it,
//            none is empty and none has more steps than a workgroup holds the scales of.
//            Prints how many plans and how many wrong ones.
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

}  // namespace

int main(int count, char** args) {
  if (count == 2 && !strcmp(args[1], "shares")) return shares();
  return 2;
}
