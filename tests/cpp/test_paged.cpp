// The paged int4 cache through the C++ API of include/turboquant.h: two sequences
// take pages, one is forked, all append and attend (decode over a shared prefix with
// a window and sinks, and a prompt), against softmax attention in double on the host;
// then a sequence ends and the pool is packed, which must not change the attention.
// With the argument "refusals": the calls that the API refuses before any GPU work.
// Exits 0 on pass.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include "turboquant.h"

using namespace turboquant;

namespace {

constexpr int kHkv = 2, kGqa = 3, kHq = kHkv * kGqa, kD = 128, kPage = 32, kPages = 24, kWidth = 6, kSeqs = 3;
constexpr int kWindow = 40, kSinks = 5;
const float kScale = 0.088388347648318447f;  // 1 / sqrt(128)
// A query is held to 2^-22 of its largest value (<= 4.5): a score of keys whose
// magnitudes add up to 0.85 D is off by 4.5 0.85 128 2^-22 / sqrt(128) = 1.1e-5,
// a weight by that of itself and 2^-17, an output by their sum times |v| <= 5.
constexpr double kTol = 1e-4;

int fails = 0;
void report(const char* what, bool ok, double err = 0.0) {
  printf("%s %s (max_err=%.3e)\n", ok ? "PASS" : "FAIL", what, err);
  fails += !ok;
}

std::mt19937 gen(77);
std::vector<float> normals(size_t n) {
  std::normal_distribution<float> nd(0.0f, 1.0f);
  std::vector<float> v(n);
  for (auto& x : v) x = nd(gen);
  return v;
}
array ints(std::vector<int32_t> v, std::vector<int64_t> shape) { return array::from_host(v.data(), shape, Dtype::int32); }
template <class T>
std::vector<T> host(const array& a) {
  std::vector<T> v(static_cast<size_t>(a.size()));
  a.to_host(v.data());
  return v;
}

// Rows [t][kvh][d] of a sequence, as the cache holds them.
struct Rows {
  std::vector<float> k, v;
};

// x [B][Hkv][T][D] quantized and back, appended to the rows of sequences `to`.
void keep(const std::vector<float>& x, int T, const std::vector<int>& to, std::vector<Rows>& seqs, bool key) {
  const int B = static_cast<int>(x.size() / (static_cast<size_t>(kHkv) * T * kD));
  const auto q = quantize(array::from_host(x.data(), {B, kHkv, T, kD}, Dtype::float32));
  const std::vector<float> y = host<float>(dequantize(q[0], q[1], q[2]));
  for (int b = 0; b < B; ++b) {
    if (to[b] < 0) continue;
    std::vector<float>& r = key ? seqs[to[b]].k : seqs[to[b]].v;
    for (int t = 0; t < T; ++t)
      for (int h = 0; h < kHkv; ++h)
        for (int d = 0; d < kD; ++d) r.push_back(y[((static_cast<size_t>(b) * kHkv + h) * T + t) * kD + d]);
  }
}

// Largest difference of out [Hq][D] from attention of q [Hq][D] at position n - 1.
double error_of(const float* out, const float* q, const Rows& r, int n, int window, int sinks) {
  double worst = 0.0;
  for (int h = 0; h < kHq; ++h) {
    const int kv = h / kGqa;
    std::vector<double> s(n, -INFINITY), ref(kD, 0.0);
    double m = -INFINITY, l = 0.0;
    for (int t = 0; t < n; ++t) {
      if (window > 0 && t < n - window && t >= sinks) continue;
      double a = 0.0;
      for (int d = 0; d < kD; ++d) a += static_cast<double>(q[h * kD + d]) * r.k[(static_cast<size_t>(t) * kHkv + kv) * kD + d];
      s[t] = a * static_cast<double>(kScale);
      m = std::max(m, s[t]);
    }
    for (int t = 0; t < n; ++t) l += s[t] == -INFINITY ? 0.0 : std::exp(s[t] - m);
    for (int t = 0; t < n; ++t) {
      if (s[t] == -INFINITY) continue;
      const double w = std::exp(s[t] - m) / l;
      for (int d = 0; d < kD; ++d) ref[d] += w * r.v[(static_cast<size_t>(t) * kHkv + kv) * kD + d];
    }
    for (int d = 0; d < kD; ++d) {
      const double e = std::fabs(ref[d] - out[h * kD + d]);
      worst = e == e ? std::max(worst, e) : INFINITY;
    }
  }
  return worst;
}

kv_pages pool(Dtype sb, void* at = nullptr) {
  const auto one = [&](int64_t last, Dtype t) {
    const std::vector<int64_t> sh = {kPages, kHkv, kPage, last};
    return at ? array::borrow(at, sh, t) : array::empty(sh, t);
  };
  return {one(kD / 8, Dtype::uint32), one(kD / 64, sb), one(kD / 64, sb),
          one(kD / 8, Dtype::uint32), one(kD / 64, sb), one(kD / 64, sb)};
}

int run() {
  kv_pages pages = pool(Dtype::float16);
  array tables = ints(std::vector<int32_t>(kSeqs * kWidth, -1), {kSeqs, kWidth});
  array refs = ints(std::vector<int32_t>(kPages, 0), {kPages});
  array lens = ints({0, 0, 0}, {kSeqs});
  std::vector<Rows> seqs(kSeqs);

  // 75 rows to sequence 0, 9 to sequence 2, in one call each
  const int T0 = 75, T2 = 9;
  report("reserve", host<int32_t>(kv_pages_reserve(tables, refs, lens, ints({T0, 0, T2}, {kSeqs}), kPage)) ==
                        std::vector<int32_t>({1, 0, 1}));
  for (int T : {T0, T2}) {
    const int to = T == T0 ? 0 : 2;
    std::vector<float> k = normals(static_cast<size_t>(kSeqs) * kHkv * T * kD), v = normals(k.size());
    std::vector<int32_t> pos(kSeqs, -1024);  // (rows outside the table are dropped)
    pos[to] = 0;
    kv_append_int4_paged(array::from_host(k.data(), {kSeqs, kHkv, T, kD}, Dtype::float32),
                         array::from_host(v.data(), {kSeqs, kHkv, T, kD}, Dtype::float32), pages, tables,
                         ints(pos, {kSeqs}));
    std::vector<int> where(kSeqs, -1);
    where[to] = to;
    keep(k, T, where, seqs, true);
    keep(v, T, where, seqs, false);
  }

  // the prompt of sequence 0: its last 50 rows attend
  {
    const int S = 50, prior = T0 - S;
    std::vector<float> q = normals(static_cast<size_t>(S) * kHq * kD);
    const std::vector<int32_t> rows = host<int32_t>(tables);
    const array table = ints(std::vector<int32_t>(rows.begin(), rows.begin() + kWidth), {kWidth});
    const auto out = host<float>(sdpa_int4_paged_prefill(array::from_host(q.data(), {S, kHq, kD}, Dtype::float32), pages,
                                                         table, prior, kGqa, kScale, kWindow, kSinks));
    double e = 0.0;
    for (int i = 0; i < S; ++i)
      e = std::max(e, error_of(&out[static_cast<size_t>(i) * kHq * kD], &q[static_cast<size_t>(i) * kHq * kD], seqs[0],
                               prior + i + 1, kWindow, kSinks));
    report("prompt", e < kTol, e);
  }

  // sequence 1 continues sequence 0 (two full pages shared), and all take a row
  lens = ints({T0, 0, T2}, {kSeqs});
  report("fork", host<int32_t>(kv_pages_fork(pages, tables, refs, lens, ints({-1, 0, -1}, {kSeqs}))) ==
                         std::vector<int32_t>({0, 1, 0}) &&
                     host<int32_t>(lens) == std::vector<int32_t>({T0, T0, T2}));
  seqs[1] = seqs[0];
  report("reserve a row", host<int32_t>(kv_pages_reserve(tables, refs, lens, ints({1, 1, 1}, {kSeqs}), kPage)) ==
                              std::vector<int32_t>({1, 1, 1}));
  {
    std::vector<float> k = normals(static_cast<size_t>(kSeqs) * kHkv * kD), v = normals(k.size());
    kv_append_int4_paged(array::from_host(k.data(), {kSeqs, kHkv, 1, kD}, Dtype::float32),
                         array::from_host(v.data(), {kSeqs, kHkv, 1, kD}, Dtype::float32), pages, tables, lens);
    keep(k, 1, {0, 1, 2}, seqs, true);
    keep(v, 1, {0, 1, 2}, seqs, false);
  }
  std::vector<int32_t> n = {T0 + 1, T0 + 1, T2 + 1};
  lens = ints(n, {kSeqs});
  std::vector<float> q = normals(static_cast<size_t>(kSeqs) * kHq * kD);
  const array Q = array::from_host(q.data(), {kSeqs, kHq, kD}, Dtype::float32);
  const auto attend = [&](const char* what, int shared, const array& windows, int window) {
    const auto out = host<float>(sdpa_int4_paged(Q, pages, tables, lens, kGqa, kScale, window, kSinks, shared, windows));
    double e = 0.0;
    for (int s = 0; s < kSeqs; ++s)
      if (n[s] > 0 && (shared == 0 || s < 2))
        e = std::max(e, error_of(&out[s * kHq * kD], &q[s * kHq * kD], seqs[s], n[s], kWindow, kSinks));
    report(what, e < kTol, e);
    return out;
  };
  const auto before = attend("decode, window and sinks", 0, {}, kWindow);
  attend("decode, a window of each sequence", 0, ints({kWindow, kWindow, kWindow}, {kSeqs}), 0);
  attend("decode over a shared prefix", 2 * kPage, {}, kWindow);

  // sequence 0 ends; the pages in use move to the front
  kv_pages_free(tables, refs, lens, ints({1, 0, 0}, {kSeqs}));
  n[0] = 0;
  const int live = host<int32_t>(kv_pages_compact(pages, tables, refs))[0];
  report("compact", live == 4 && host<int32_t>(lens) == n);  // sequence 1: 3 pages, 2: one
  const auto after = attend("decode after packing", 0, {}, kWindow);
  report("packing changes nothing", std::memcmp(&before[kHq * kD], &after[kHq * kD], 2 * kHq * kD * sizeof(float)) == 0);

  // a page copied elsewhere and read there
  auto t = host<int32_t>(tables);
  const int32_t src = t[2 * kWidth], dst = kPages - 1;
  kv_pages_copy(pages, ints({src}, {1}), ints({dst}, {1}));
  t[2 * kWidth] = dst;
  tables = ints(t, {kSeqs, kWidth});
  attend("decode from a copied page", 0, {}, kWindow);

  // evicted: sequence 1's second page lies in rows 32 .. 63 of 76, none of it behind
  // sinks and before a window of 10 stays
  t[2 * kWidth] = src;
  tables = ints(t, {kSeqs, kWidth});
  kv_pages_evict(tables, refs, lens, kPage, 10, kSinks);
  const auto left = host<int32_t>(tables);
  report("evict", left[kWidth] == t[kWidth] && left[kWidth + 1] == -1 && left[kWidth + 2] == t[kWidth + 2] &&
                      left[2 * kWidth] == src);
  return fails;
}

template <class F>
void refused(const char* what, F f) {
  bool ok = false;
  try {
    f();
  } catch (const std::exception& e) {
    ok = e.what()[0] != 0;
    printf("%s\n", e.what());
  }
  report(what, ok);
}

int refusals() {
  alignas(16) static char here[64];
  const auto at = [&](std::vector<int64_t> sh, Dtype t) { return array::borrow(here, std::move(sh), t); };
  kv_pages p = pool(Dtype::float16, here);
  array tables = at({kSeqs, kWidth}, Dtype::int32), lens = at({kSeqs}, Dtype::int32), refs = at({kPages}, Dtype::int32);
  const array k = at({kSeqs, kHkv, 1, kD}, Dtype::float32), q = at({kSeqs, kHq, kD}, Dtype::float32);
  const array fl = at({kSeqs}, Dtype::float32);
  refused("append: rows of another head_dim", [&] { kv_append_int4_paged(at({kSeqs, kHkv, 1, 256}, Dtype::float32), at({kSeqs, kHkv, 1, 256}, Dtype::float32), p, tables, lens); });
  refused("append: k and v of different types", [&] { kv_append_int4_paged(k, at({kSeqs, kHkv, 1, kD}, Dtype::float16), p, tables, lens); });
  refused("append: positions not int32", [&] { kv_append_int4_paged(k, k, p, tables, fl); });
  refused("append: another batch than the tables'", [&] { kv_append_int4_paged(k, k, p, at({kSeqs + 1, kWidth}, Dtype::int32), lens); });
  kv_pages odd = p;
  odd.v_biases = at({kPages, kHkv, kPage, kD / 64}, Dtype::float32);
  refused("pages of two scale types", [&] { kv_append_int4_paged(k, k, odd, tables, lens); });
  odd = p;
  odd.v_quant = at({kPages, kHkv, kPage, kD / 4}, Dtype::uint32);
  refused("pages of two widths", [&] { kv_append_int4_paged(k, k, odd, tables, lens); });
  refused("decode: queries of another batch", [&] { sdpa_int4_paged(at({kSeqs + 1, kHq, kD}, Dtype::float32), p, tables, lens, kGqa); });
  refused("decode: tables of one axis", [&] { sdpa_int4_paged(q, p, lens, lens, kGqa); });
  refused("prompt: a table of two axes", [&] { sdpa_int4_paged_prefill(q, p, tables, 0, kGqa); });
  refused("fork: refs of another pool", [&] {
    array few = at({kPages - 1}, Dtype::int32);
    kv_pages_free(tables, few, lens, at({kSeqs + 1}, Dtype::int32));
  });
  refused("free: lengths not int32", [&] {
    array l = fl;
    kv_pages_free(tables, refs, l, lens);
  });
  refused("evict: no window", [&] { kv_pages_evict(tables, refs, lens, kPage, 0); });
  refused("evict: a page size that is no power of two", [&] { kv_pages_evict(tables, refs, lens, 48, 10); });
  refused("compact: refs of another pool", [&] {
    array few = at({kPages - 1}, Dtype::int32);
    kv_pages_compact(p, tables, few);
  });
  refused("copy: src and dst of different counts", [&] { kv_pages_copy(p, at({2}, Dtype::int32), at({3}, Dtype::int32)); });
  return fails;
}

}  // namespace

int main(int argc, char** argv) { return (argc > 1 && std::string(argv[1]) == "refusals" ? refusals() : run()) == 0 ? 0 : 1; }
