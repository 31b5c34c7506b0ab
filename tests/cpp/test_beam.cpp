// Beam search and batched chunks through include/turboquant.h.  With the argument
// "refusals": calls that are refused before any GPU work, each by the message of its own
// check.  Without: a run of the calls against the host.  Exits 0 on pass.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <random>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "turboquant.h"

using namespace turboquant;

namespace {

constexpr int kHkv = 2, kGqa = 3, kHq = kHkv * kGqa, kD = 128, kPage = 32, kPages = 24, kWidth = 4, kSeqs = 3;

int fails = 0;

template <class F>
void refused(const char* what, const char* message, F f) {
  std::string got = "no exception";
  try {
    f();
  } catch (const std::exception& e) {
    got = e.what();
  }
  const bool ok = got.find(message) != std::string::npos;
  printf("%s %s: %s\n", ok ? "PASS" : "FAIL", what, got.c_str());
  fails += !ok;
}

template <class T>
std::vector<T> host(const array& a) {
  std::vector<T> v(static_cast<size_t>(a.size()));
  a.to_host(v.data());
  return v;
}
array ints(std::vector<int32_t> v, std::vector<int64_t> shape) { return array::from_host(v.data(), shape, Dtype::int32); }

void report(const char* what, bool ok) {
  printf("%s %s\n", ok ? "PASS" : "FAIL", what);
  fails += !ok;
}

int run() {
  std::mt19937 gen(5);
  std::normal_distribution<float> nd(0.0f, 1.0f);
  const auto normals = [&](std::vector<int64_t> shape) {
    size_t n = 1;
    for (int64_t d : shape) n *= static_cast<size_t>(d);
    std::vector<float> v(n);
    for (float& x : v) x = nd(gen);
    return array::from_host(v.data(), shape, Dtype::float32);
  };

  // the five best of three beams of 2,000 tokens
  const int W = 3, V = 2000, K = 5;
  const array x = normals({1, W, V});
  std::vector<float> scores = {-1.0f, -0.5f, -3.0f};
  const beams b = beam_select(x, array::from_host(scores.data(), {1, W}, Dtype::float32), K);
  const std::vector<float> hx = host<float>(x);
  std::vector<std::pair<double, int>> all;
  for (int w = 0; w < W; ++w) {
    double sum = 0.0;
    for (int t = 0; t < V; ++t) sum += std::exp(static_cast<double>(hx[w * V + t]));
    for (int t = 0; t < V; ++t) all.push_back({-(scores[w] + hx[w * V + t] - std::log(sum)), w * V + t});
  }
  std::sort(all.begin(), all.end());
  bool same = true;
  const auto got = host<float>(b.scores);
  const auto parents = host<int32_t>(b.parents), tokens = host<int32_t>(b.tokens);
  for (int k = 0; k < K; ++k)
    same = same && parents[k] * V + tokens[k] == all[k].second && std::fabs(got[k] + all[k].first) < 1e-5;
  report("beam_select", same);

  // pages: sequence 1 becomes a second child of 0 (one page shared, one copied), 0 stays
  const auto one = [&](int64_t last, Dtype t) { return array::empty({kPages, kHkv, kPage, last}, t); };
  kv_pages p{one(kD / 8, Dtype::uint32), one(kD / 64, Dtype::float16), one(kD / 64, Dtype::float16),
             one(kD / 8, Dtype::uint32), one(kD / 64, Dtype::float16), one(kD / 64, Dtype::float16)};
  array tables = ints({3, 9, 1, -1, 4, -1, -1, -1}, {2, 4});
  std::vector<int32_t> counts(kPages, 0);
  for (int e : {3, 9, 1, 4}) counts[e] = 1;
  array refs = ints(counts, {kPages}), lens = ints({90, 20}, {2});
  kv_append_int4_paged(normals({2, kHkv, 90, kD}), normals({2, kHkv, 90, kD}), p, tables, ints({0, 0}, {2}));
  report("kv_pages_reorder", host<int32_t>(kv_pages_reorder(p, tables, refs, lens, ints({0, 0}, {2}))) == std::vector<int32_t>({1, 1}) &&
                                 host<int32_t>(tables) == std::vector<int32_t>({3, 9, 1, -1, 3, 9, 0, -1}) &&
                                 host<int32_t>(lens) == std::vector<int32_t>({90, 90}));

  // both sequences' last 5 queries: as a prompt's of one sequence
  const array q = normals({10, kHq, kD});
  const auto chunks = host<float>(sdpa_int4_paged_chunks(q, p, tables, ints({0, 5, 10}, {3}), lens, kGqa, 0.09f));
  bool near = true;
  for (int s = 0; s < 2; ++s) {
    const array mine = array::borrow(const_cast<char*>(static_cast<const char*>(q.data())) + s * 5 * kHq * kD * 4, {5, kHq, kD}, Dtype::float32);
    const auto want = host<float>(sdpa_int4_paged_prefill(mine, p, ints({3, 9, s == 0 ? 1 : 0, -1}, {4}), 85, kGqa, 0.09f));
    for (size_t i = 0; i < want.size(); ++i) near = near && std::fabs(want[i] - chunks[s * want.size() + i]) < 1e-4f;
  }
  report("sdpa_int4_paged_chunks", near);

  // a contiguous cache: two sequences change places
  const auto cache = [&](int64_t last, Dtype t) { return array::empty({2, kHkv, 50, last}, t); };
  array c[6] = {cache(kD / 8, Dtype::uint32), cache(kD / 64, Dtype::float16), cache(kD / 64, Dtype::float16),
                cache(kD / 8, Dtype::uint32), cache(kD / 64, Dtype::float16), cache(kD / 64, Dtype::float16)};
  kv_append_int4(normals({2, kHkv, 50, kD}), normals({2, kHkv, 50, kD}), c[0], c[1], c[2], c[3], c[4], c[5], ints({0, 0}, {2}));
  const auto before = host<uint32_t>(c[3]);
  array n = ints({50, 50}, {2});
  kv_reorder_int4(c[0], c[1], c[2], c[3], c[4], c[5], n, ints({1, 0}, {2}));
  auto after = host<uint32_t>(c[3]);
  std::rotate(after.begin(), after.begin() + after.size() / 2, after.end());
  report("kv_reorder_int4", after == before && host<int32_t>(n) == std::vector<int32_t>({50, 50}));
  return fails;
}

}  // namespace

int main(int argc, char** argv) {
  if (argc < 2 || std::string(argv[1]) != "refusals") return run() == 0 ? 0 : 1;
  alignas(16) static char here[64];  // never read
  const auto at = [&](std::vector<int64_t> sh, Dtype t) { return array::borrow(here, std::move(sh), t); };
  const auto i32 = [&](std::vector<int64_t> sh) { return at(std::move(sh), Dtype::int32); };
  const auto f32 = [&](std::vector<int64_t> sh) { return at(std::move(sh), Dtype::float32); };
  const auto one = [&](int64_t last, Dtype t) { return at({kPages, kHkv, kPage, last}, t); };
  kv_pages p{one(kD / 8, Dtype::uint32), one(kD / 64, Dtype::float16), one(kD / 64, Dtype::float16),
             one(kD / 8, Dtype::uint32), one(kD / 64, Dtype::float16), one(kD / 64, Dtype::float16)};
  array tables = i32({kSeqs, kWidth}), lens = i32({kSeqs}), refs = i32({kPages}), few = i32({kPages - 1}), none = i32({kSeqs + 1});
  const array q = f32({5, kHq, kD}), x = f32({2, 4, 100}), sc = f32({2, 4});

  refused("chunks: starts of another batch", "starts: int32 of another shape", [&] { sdpa_int4_paged_chunks(q, p, tables, lens, lens, kGqa); });
  refused("chunks: lengths of another batch", "seq_lens: int32 of another shape", [&] { sdpa_int4_paged_chunks(q, p, tables, none, none, kGqa); });
  refused("chunks: queries of another head_dim", "queries must be", [&] { sdpa_int4_paged_chunks(f32({5, kHq, 64}), p, tables, none, lens, kGqa); });
  refused("chunks: tables of one axis", "block_tables must be int32", [&] { sdpa_int4_paged_chunks(q, p, lens, none, lens, kGqa); });
  refused("reorder: refs of another pool", "refs: int32 of another shape", [&] { kv_pages_reorder(p, tables, few, lens, lens); });
  refused("reorder: parents of another batch", "parents: int32 of another shape", [&] { kv_pages_reorder(p, tables, refs, lens, none); });
  refused("reorder: lengths of another batch", "lengths: int32 of another shape", [&] { kv_pages_reorder(p, tables, refs, none, lens); });
  refused("select: logits of two axes", "logits must be", [&] { beam_select(sc, sc); });
  refused("select: scores of another batch", "scores must be", [&] { beam_select(x, f32({2, 3})); });
  refused("select: scores not float32", "scores must be", [&] { beam_select(x, i32({2, 4})); });
  refused("select: finished not uint8", "finished must be", [&] { beam_select(x, sc, 4, i32({2, 4})); });
  refused("select: no results", "num_out must be", [&] { beam_select(x, sc, -1); });
  refused("rows: parents of another batch", "parents: int32 of another shape", [&] {
    array n = i32({kPages}), from = i32({3});
    kv_reorder_int4(p.k_quant, p.k_scales, p.k_biases, p.v_quant, p.v_scales, p.v_biases, n, from);
  });
  refused("rows: scales of another width", "scales / biases must be", [&] {
    array n = i32({kPages}), odd = at({kPages, kHkv, kPage, 1}, Dtype::float16);
    kv_reorder_int4(p.k_quant, odd, p.k_biases, p.v_quant, p.v_scales, p.v_biases, n, n);
  });
  printf("%d failed\n", fails);
  return fails == 0 ? 0 : 1;
}
