// Calls of the paged cache of include/turboquant.h.  With the argument "refusals":
// those that are refused before any GPU work, each by the message of its own check (what
// a call without that check throws, at its first GPU call where there is no GPU, is
// another one).  Without: rows are counted only where they have pages, and a shared
// prefix is read by a table of its own.  Exits 0 on pass.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include "turboquant.h"

using namespace turboquant;

namespace {

constexpr int kHkv = 2, kGqa = 3, kHq = kHkv * kGqa, kD = 128, kPage = 32, kPages = 24, kWidth = 6, kSeqs = 3;

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
  // two sequences of two shared pages and one of their own
  const auto one = [&](int64_t last, Dtype t) { return array::empty({kPages, kHkv, kPage, last}, t); };
  kv_pages p{one(kD / 8, Dtype::uint32), one(kD / 64, Dtype::float16), one(kD / 64, Dtype::float16),
             one(kD / 8, Dtype::uint32), one(kD / 64, Dtype::float16), one(kD / 64, Dtype::float16)};
  const std::vector<int32_t> rows = {3, 9, 1, 7, 3, 9, 4, -1};
  array tables = ints(rows, {2, 4}), refs = ints(std::vector<int32_t>(kPages, 0), {kPages});
  std::mt19937 gen(5);
  std::normal_distribution<float> nd(0.0f, 1.0f);
  const auto normals = [&](std::vector<int64_t> shape) {
    size_t n = 1;
    for (int64_t d : shape) n *= static_cast<size_t>(d);
    std::vector<float> v(n);
    for (float& x : v) x = nd(gen);
    return array::from_host(v.data(), shape, Dtype::float32);
  };
  const array first = ints({0}, {1}), t0 = ints({3, 9, 1, 7}, {1, 4}), t1 = ints({3, 9, 4, -1}, {1, 4});
  kv_append_int4_paged(normals({1, kHkv, 128, kD}), normals({1, kHkv, 128, kD}), p, t0, first);
  kv_append_int4_paged(normals({1, kHkv, 96, kD}), normals({1, kHkv, 96, kD}), p, t1, first);

  array lens = ints({90, 90}, {2});
  report("advance", host<int32_t>(kv_pages_advance(tables, refs, lens, ints({7, 7}, {2}), kPage)) == std::vector<int32_t>({1, 0}) &&
                        host<int32_t>(lens) == std::vector<int32_t>({97, 90}));

  const array q = normals({2, kHq, kD});
  const auto want = host<float>(sdpa_int4_paged(q, p, tables, lens, kGqa, 0.09f, 0, 0, 2 * kPage));
  report("attention is finite", std::all_of(want.begin(), want.end(), [](float x) { return std::isfinite(x); }));
  const array lost = ints({-1, -1, 1, 7, 3, 9, 4, -1}, {2, 4});
  const auto got = host<float>(sdpa_int4_paged(q, p, lost, lens, kGqa, 0.09f, 0, 0, 2 * kPage, {}, -1, {}, ints({3, 9}, {2})));
  report("a prefix by its own table", got == want);
  return fails;
}

}  // namespace

int main(int argc, char** argv) {
  if (argc < 2 || std::string(argv[1]) != "refusals") return run() == 0 ? 0 : 1;
  alignas(16) static char here[64];  // never read
  const auto at = [&](std::vector<int64_t> sh, Dtype t) { return array::borrow(here, std::move(sh), t); };
  const auto i32 = [&](std::vector<int64_t> sh) { return at(std::move(sh), Dtype::int32); };
  const auto f32 = [&](std::vector<int64_t> sh) { return at(std::move(sh), Dtype::float32); };
  const auto pool = [&](std::vector<int64_t> sh) {
    const auto one = [&](int64_t last, Dtype t) {
      std::vector<int64_t> x = sh;
      x.push_back(last);
      return at(x, t);
    };
    return kv_pages{one(kD / 8, Dtype::uint32), one(kD / 64, Dtype::float16), one(kD / 64, Dtype::float16),
                    one(kD / 8, Dtype::uint32), one(kD / 64, Dtype::float16), one(kD / 64, Dtype::float16)};
  };
  kv_pages p = pool({kPages, kHkv, kPage}), layered = pool({2, kPages, kHkv, kPage});
  array tables = i32({kSeqs, kWidth}), lens = i32({kSeqs}), refs = i32({kPages}), few = i32({kPages - 1});
  const array k = f32({kSeqs, kHkv, 1, kD}), q = f32({kSeqs, kHq, kD}), none = i32({kSeqs + 1});
  array fl = f32({kSeqs});

  refused("append: rows of another head_dim", "do not fit the pages", [&] { kv_append_int4_paged(f32({kSeqs, kHkv, 1, 256}), f32({kSeqs, kHkv, 1, 256}), p, tables, lens); });
  refused("append: another batch than the tables'", "do not fit the pages", [&] { kv_append_int4_paged(k, k, p, i32({kSeqs + 1, kWidth}), lens); });
  refused("append: k and v of different types", "of one dtype", [&] { kv_append_int4_paged(k, at({kSeqs, kHkv, 1, kD}, Dtype::float16), p, tables, lens); });
  refused("append: positions not int32", "positions: int32", [&] { kv_append_int4_paged(k, k, p, tables, fl); });
  refused("append: positions of another batch", "positions: int32", [&] { kv_append_int4_paged(k, k, p, tables, none); });
  refused("append: tables not int32", "block_tables must be int32", [&] { kv_append_int4_paged(k, k, p, f32({kSeqs, kWidth}), lens); });
  refused("append: pages of layers", "pages must be", [&] { kv_append_int4_paged(k, k, layered, tables, lens); });
  kv_pages odd = p;
  odd.v_biases = f32({kPages, kHkv, kPage, kD / 64});
  refused("pages of two scale types", "of one dtype", [&] { kv_append_int4_paged(k, k, odd, tables, lens); });
  odd = p;
  odd.v_quant = at({kPages, kHkv, kPage, kD / 4}, Dtype::uint32);
  refused("pages of two widths", "uint32 of one shape", [&] { kv_append_int4_paged(k, k, odd, tables, lens); });
  odd = p;
  odd.k_scales = at({kPages, kHkv, kPage, 1}, Dtype::float16);
  refused("scales of another width", "scales / biases must be", [&] { kv_append_int4_paged(k, k, odd, tables, lens); });

  refused("decode: queries of another batch", "queries must be", [&] { sdpa_int4_paged(f32({kSeqs + 1, kHq, kD}), p, tables, lens, kGqa); });
  refused("decode: tables of one axis", "block_tables must be int32", [&] { sdpa_int4_paged(q, p, lens, lens, kGqa); });
  refused("decode: lengths of another batch", "seq_lens: int32 of another shape", [&] { sdpa_int4_paged(q, p, tables, none, kGqa); });
  refused("decode: windows not int32", "windows: int32 of another shape", [&] { sdpa_int4_paged(q, p, tables, lens, kGqa, 1.0f, 0, 0, 0, fl); });
  refused("decode: a prefix's table of another length", "prefix_table: int32 of another shape", [&] { sdpa_int4_paged(q, p, tables, lens, kGqa, 1.0f, 0, 0, kPage, {}, -1, {}, i32({2})); });
  refused("prompt: a table of two axes", "block_table must be int32 (max_pages)", [&] { sdpa_int4_paged_prefill(q, p, tables, 0, kGqa); });
  refused("prompt: queries of another head_dim", "queries must be", [&] { sdpa_int4_paged_prefill(f32({5, kHq, 64}), p, lens, 0, kGqa); });

  refused("reserve: tables not int32", "block_tables must be int32", [&] { array t = f32({kSeqs, kWidth}); kv_pages_reserve(t, refs, lens, lens, kPage); });
  refused("reserve: refs of two axes", "refs must be int32", [&] { kv_pages_reserve(tables, tables, lens, lens, kPage); });
  refused("reserve: lengths of another batch", "lengths: int32 of another shape", [&] { kv_pages_reserve(tables, refs, none, lens, kPage); });
  refused("reserve: requests not int32", "n_new: int32 of another shape", [&] { kv_pages_reserve(tables, refs, lens, fl, kPage); });
  refused("advance: counts of another batch", "n_new: int32 of another shape", [&] { kv_pages_advance(tables, refs, lens, none, kPage); });
  refused("advance: refs not int32", "refs must be int32", [&] { kv_pages_advance(tables, fl, lens, lens, kPage); });
  refused("fork: pages of three axes", "pages must be", [&] { kv_pages o = pool({kPages, kHkv}); kv_pages_fork(o, tables, refs, lens, lens); });
  refused("fork: refs of another pool", "refs: int32 of another shape", [&] { kv_pages_fork(p, tables, few, lens, lens); });
  refused("fork: lengths of another batch", "lengths: int32 of another shape", [&] { array l = i32({kSeqs + 1}); kv_pages_fork(p, tables, refs, l, lens); });
  refused("fork: parents of another batch", "parents: int32 of another shape", [&] { kv_pages_fork(p, tables, refs, lens, none); });
  refused("free: lengths not int32", "lengths: int32 of another shape", [&] { kv_pages_free(tables, refs, fl, lens); });
  refused("free: another batch", "which: int32 of another shape", [&] { kv_pages_free(tables, refs, lens, none); });
  refused("evict: no window", "sliding_window must be > 0", [&] { kv_pages_evict(tables, refs, lens, kPage, 0); });
  refused("evict: a page size that is no power of two", "page_size must be a power of two", [&] { kv_pages_evict(tables, refs, lens, 48, 10); });
  refused("evict: another batch", "which: int32 of another shape", [&] { kv_pages_evict(tables, refs, lens, kPage, 10, 0, none); });
  refused("compact: refs of another pool", "refs: int32 of another shape", [&] { kv_pages_compact(p, tables, few); });
  refused("copy: src and dst of different counts", "dst: int32 of another shape", [&] { kv_pages_copy(p, i32({2}), i32({3})); });
  refused("copy: src of two axes", "src must be int32 (n)", [&] { kv_pages_copy(p, tables, tables); });
  printf("%d failed\n", fails);
  return fails == 0 ? 0 : 1;
}
