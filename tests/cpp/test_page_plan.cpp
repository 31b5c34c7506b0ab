// The sums of a page plan (csrc/tq_page_plan.h) on the host: requests are granted in
// order as long as the free pages last, also where all requests together need more
// pages than 32 bits count.  Exits 0 on pass.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <random>
#include <vector>

#include "../../gemma4metal_amd/csrc/tq_page_plan.h"

using namespace tq;

namespace {

int fails = 0;

// As pages_plan_kernel: scans of 1,024 sequences, their sums carried on.
std::vector<int> granted(const std::vector<int>& need, int num_pages, int found) {
  constexpr size_t kTile = 1024;
  std::vector<int> out(need.size());
  PlanSum want = 0;
  for (size_t s0 = 0; s0 < need.size(); s0 += kTile) {
    PlanSum b = 0;
    for (size_t s = s0; s < std::min(need.size(), s0 + kTile); ++s) {
      out[s] = plan_grants(need[s], plan_before(want + b, num_pages), found);
      b += std::max(need[s], 0);
    }
    want += b;
  }
  return out;
}

bool right(const std::vector<int>& need, int num_pages, int found) {
  std::vector<int> ref(need.size());
  __int128 before = 0;
  for (size_t s = 0; s < need.size(); ++s) {
    ref[s] = need[s] == 0 || (need[s] > 0 && before + need[s] <= found);
    before += std::max(need[s], 0);
  }
  return granted(need, num_pages, found) == ref;
}

void report(const char* what, bool ok) {
  printf("%s %s\n", ok ? "PASS" : "FAIL", what);
  fails += !ok;
}

}  // namespace

int main() {
  constexpr int kRow = (1 << 26) - (1 << 11), kPool = 1 << 28;  // pages of a sequence, of a pool
  std::vector<int> big(34, kRow);
  big.insert(big.end(), {1, 0, -1, 5, 1});
  report("34 sequences that need 2^31 pages", right(big, 5, 5));
  report("the same, the largest pool", right(big, kPool, kPool));
  report("1,024 of them, the largest pool", right(std::vector<int>(1024, kRow), kPool, kPool));
  report("65 scans, sums past 2^42", right(std::vector<int>(65 * 1024, kRow), kPool, kPool - 3));
  std::vector<int> wrap(64, 1 << 26);  // 2^32 in all: 0 in 32 bits
  wrap.push_back(1);
  report("a sum that is 0 in 32 bits", right(wrap, 100, 100));
  std::mt19937 gen(3);
  bool small = true;
  for (int round = 0; round < 200; ++round) {
    std::vector<int> need(1 + gen() % 3000);
    for (int& n : need) n = static_cast<int>(gen() % 7) - 1;
    const int pages = 1 + static_cast<int>(gen() % 4000);
    small &= right(need, pages, static_cast<int>(gen() % (pages + 1)));
  }
  report("small requests", small);
  return fails == 0 ? 0 : 1;
}
