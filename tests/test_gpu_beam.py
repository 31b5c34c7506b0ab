"""GPU: beam search over the int4 KV cache -- the choice of beams, the reordering of
pages and of contiguous caches -- against the oracle."""
import itertools

import numpy as np
import pytest
import torch

from oracle import beam as OB
from oracle import oracle as O
from oracle import paged as OP
from tests.gpu_util import dev, host, queries
from tests.test_gpu_paged import ints

pytestmark = pytest.mark.gpu

EPS32 = 2.0**-24


@pytest.fixture(scope="module")
def bm():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from gemma4metal_amd import beam
    return beam


@pytest.fixture(scope="module")
def pg():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from gemma4metal_amd import paged
    return paged


_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def logits(rng, shape, dtype):
    t = torch.from_numpy((3 * rng.standard_normal(shape)).astype(np.float32)).to(_DT[dtype]).cuda()
    return t, t.float().cpu().numpy()


def near(got, x, scores, val, K):
    """Unlike beams' candidates may change places where their totals differ by less
    than the two logs' errors (see check), 2 (21 + 3 35 + 2) 2^-24 = 1.6e-5; a beam's
    own come in their order, none left out."""
    B, W, V = x.shape
    parents, tokens = host(got[1]), host(got[2])
    for b in range(B):
        t = OB.totals(x[b], scores[b], None, 0)
        w = parents[b] - b * W
        assert np.abs(t[w, tokens[b]] - val[b]).max() <= 2 * 128 * EPS32
        for i in range(W):
            mine = tokens[b][w == i]
            assert np.array_equal(mine, np.argsort(-t[i], kind="stable")[:len(mine)])


def check(got, x, scores, K, finished=None, pad=0, exact=True):
    val, parents, tokens = OB.beam_select(x, scores, K, finished, pad)
    if exact:
        assert np.array_equal(host(got[1]), parents)
        assert np.array_equal(host(got[2]), tokens)
    else:
        near(got, x, scores, val, K)
    s = host(got[0]).astype(np.float64)
    assert s.shape == val.shape and np.array_equal(np.isfinite(s), np.isfinite(val))
    fine = np.isfinite(val)
    # the total's rounding, and of the log of the sum: 16 terms a lane and six steps
    # (at most 21 roundings), each exponential off by its argument's roundings (three
    # of at most 24 log2 e) and an ulp
    bound = EPS32 * (np.abs(val[fine]) + 21 + 3 * 35 + 2)
    assert np.all(np.abs(s[fine] - val[fine]) <= bound)
    assert np.array_equal(s[~fine], val[~fine])


# ---------------------------------------------------------------------------
# choosing
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,W,V,K", [(1, 1, 1, 1), (1, 2, 3, 64), (2, 4, 1000, 4), (3, 5, 1024, 10), (2, 3, 1025, 3),
                                     (1, 64, 2049, 64), (2, 7, 5003, 16), (1, 4, 70001, 17), (5, 1, 4096, 8)])
def test_select(bm, dtype, B, W, V, K):
    rng = np.random.default_rng(V + K)
    x, xf = logits(rng, (B, W, V), dtype)
    scores = (-20 * rng.random((B, W))).astype(np.float32)
    check(bm.beam_select(x, dev(scores), K), xf, scores, K)


def test_a_vocabulary_of_more_sums_than_lanes(bm):
    rng = np.random.default_rng(13)
    x, xf = logits(rng, (1, 2, 300001), "bf16")
    scores = np.array([[-1.0, -1.25]], np.float32)
    check(bm.beam_select(x, dev(scores), 5), xf, scores, 5)


def test_ties_go_to_the_lowest(bm):
    """Equal rows at unlike alignments, equal logits, and rows of one value."""
    rng = np.random.default_rng(3)
    x, xf = logits(rng, (2, 1, 3001), "bf16")
    x, xf = x.expand(2, 5, 3001).contiguous(), np.repeat(xf, 5, 1)
    scores = np.zeros((2, 5), np.float32)
    check(bm.beam_select(x, dev(scores), 12), xf, scores, 12)
    few = rng.integers(0, 3, (2, 4, 5000)).astype(np.float32)
    scores = np.full((2, 4), -1.5, np.float32)
    for K in (1, 16, 64):
        check(bm.beam_select(dev(few), dev(scores), K), few, scores, K)
    flat = np.zeros((1, 3, 9000), np.float32)
    check(bm.beam_select(dev(flat), dev(scores[:1, :3].copy()), 64), flat, scores[:1, :3], 64)


def test_strided_logits(bm):
    rng = np.random.default_rng(4)
    x, xf = logits(rng, (3, 4, 2100), "f16")
    scores = (-5 * rng.random((3, 4))).astype(np.float32)
    check(bm.beam_select(x[:, :, :2053], dev(scores), 6), xf[:, :, :2053], scores, 6)
    check(bm.beam_select(x[:, :, 3:], dev(scores), 6), xf[:, :, 3:], scores, 6)
    t = x.transpose(0, 1)
    check(bm.beam_select(t, dev(scores.T.copy()), 6), xf.transpose(1, 0, 2), scores.T, 6)
    check(bm.beam_select(x[:, :1].expand(3, 4, 2100), dev(scores), 6), np.repeat(xf[:, :1], 4, 1), scores, 6)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_tokens(bm, dtype):
    """Tokens of -inf, of the type's lowest value, NaN and +inf; beams without any
    token; fewer candidates than asked for."""
    rng = np.random.default_rng(6)
    W, V = 6, 4100
    x, _ = logits(rng, (2, W, V), dtype)
    low = torch.finfo(_DT[dtype]).min
    x[0, 0, :] = -np.inf                      # no token
    x[0, 1, 1:] = -np.inf                     # one token
    x[0, 2, :] = low                          # all alike
    x[0, 3, 5:4000] = low                     # masked by the lowest value
    x[0, 4, ::3] = float("nan")
    x[0, 5, [7, 4099]] = np.inf               # two share the probability
    x[1, :, :] = -np.inf
    x[1, 2, 4097:] = 1.0
    x[1, 4, 1024:1030] = float("nan")
    xf = x.float().cpu().numpy()
    scores = (-rng.random((2, W))).astype(np.float32)
    for K in (3, 64):
        check(bm.beam_select(x, dev(scores), K), xf, scores, K)


def test_finished_and_dead_beams(bm):
    rng = np.random.default_rng(8)
    B, W, V = 3, 4, 2500
    x, xf = logits(rng, (B, W, V), "bf16")
    x[0, 1] = float("nan")                    # a finished beam's logits are not looked at
    scores = (-3 * rng.random((B, W))).astype(np.float32)
    scores[1, 1:] = -np.inf                   # a request's first step
    scores[2, 0] = np.nan
    done = np.zeros((B, W), bool)
    done[0, 1] = done[2, 2] = True
    scores[2, 2] = 0.5
    done[2, 1] = True
    scores[2, 1] = -np.inf
    for K, pad in ((4, 0), (9, 2400)):
        check(bm.beam_select(x, dev(scores), K, finished=torch.from_numpy(done).cuda(), pad_token=pad), xf, scores, K,
              done, pad)
    every = np.ones((B, W), bool)
    got = bm.beam_select(x, dev(scores), 4, finished=torch.from_numpy(every).cuda(), pad_token=7)
    check(got, xf, scores, 4, every, 7)


def test_candidates_that_crowd(bm):
    """More of them than are kept at once: few tokens allowed, the same ones in every
    segment, and 64 wanted."""
    rng = np.random.default_rng(9)
    x = np.full((1, 8, 64 * 1024), -np.inf, np.float32)
    for j in range(64):
        x[0, :, j * 1024:j * 1024 + 48] = rng.standard_normal((8, 48))
    scores = np.zeros((1, 8), np.float32)
    check(bm.beam_select(dev(x), dev(scores), 64), x, scores, 64)
    up = np.linspace(-9, 9, 2 * 40000, dtype=np.float32).reshape(1, 2, 40000)
    # (the rows are one another's in turn, but for their rounding: totals differ by 1e-8)
    check(bm.beam_select(dev(up), dev(scores[:, :2].copy()), 64), up, scores[:, :2], 64, exact=False)


def test_select_in_a_graph_and_on_a_stream(bm):
    rng = np.random.default_rng(10)
    x, _ = logits(rng, (2, 4, 30000), "bf16")
    scores = dev((-rng.random((2, 4))).astype(np.float32))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bm.beam_select(x, scores)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = bm.beam_select(x, scores)
    for i in range(3):
        x.copy_(logits(rng, (2, 4, 30000), "bf16")[0])
        g.replay()
        torch.cuda.synchronize()
        check(got, x.float().cpu().numpy(), host(scores), 4)
        eager = bm.beam_select(x, scores, stream=s)
        s.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


# ---------------------------------------------------------------------------
# reordering pages
# ---------------------------------------------------------------------------

def pool_of(rng, S, width, N, page, lens, share=0, layers=2, Hkv=1, D=64):
    """A pool whose sequences have the pages of their lengths; the first `share` full
    ones are sequence 0's for all."""
    tables, refs = np.full((S, width), -1, np.int32), np.zeros(N, np.int32)
    order = iter(rng.permutation(N))
    for s in range(S):
        for e in range(-(-lens[s] // page)):
            p = tables[0, e] if s and e < share and e < lens[s] // page and e < lens[0] // page else next(order)
            tables[s, e] = p
            refs[p] += 1
    lead = (layers, N, Hkv, page)
    pages = [rng.integers(0, 2**32, lead + (D // 8,), dtype=np.uint32) if i % 3 == 0
             else rng.standard_normal(lead + (D // 64,)).astype(np.float16) for i in range(6)]
    return OP.Pool(tables, refs, np.array(lens, np.int32), page, pages)


def run_reorder(pg, pool, parents, **kw):
    pages = [dev(p) for p in pool.pages]
    t, r, n = dev(pool.tables), dev(pool.refs), dev(pool.lengths)
    got = host(pg.kv_pages_reorder(pages, t, r, n, ints(parents), **kw))
    want = OB.reorder(pool, parents)
    assert np.array_equal(got, want)
    assert np.array_equal(host(n), pool.lengths)
    assert np.array_equal(host(t), pool.tables)
    assert np.array_equal(host(r), pool.refs)
    for a, b in zip(pages, pool.pages):
        assert np.array_equal(host(a), b)
    return want


def counted(pool):
    refs = np.zeros_like(pool.refs)
    for e in pool.tables.ravel():
        if pool._is_page(e):
            refs[e] += 1
    return refs


@pytest.mark.parametrize("S,page,lo,hi", [(1, 32, 0, 70), (2, 32, 1, 40), (5, 64, 60, 70), (8, 32, 31, 33),
                                          (12, 128, 0, 500), (300, 32, 1, 100)])
def test_reorder_pages(pg, S, page, lo, hi):
    rng = np.random.default_rng(S)
    lens = rng.integers(lo, hi + 1, S).tolist()
    width = hi // page + 2
    for share in (0, 1):
        pool = pool_of(rng, S, width, S * width + 2, page, lens, share)
        for _ in range(3):
            parents = rng.integers(0, S, S)
            parents[rng.random(S) < 0.1] = -1
            run_reorder(pg, pool, parents)
            assert np.array_equal(counted(pool), pool.refs)


@pytest.mark.parametrize("S,width", [(256, 16), (256, 17), (257, 3), (64, 64), (8, 512), (8, 513), (1, 4096), (1, 5000)])
def test_reorder_pages_of_many_entries(pg, S, width):
    """Few and many sequences and table entries, on both sides of where the plan takes
    the roles too."""
    rng = np.random.default_rng(S + width)
    lens = rng.integers(1, 32 * min(width, 40), S).tolist()
    pool = pool_of(rng, S, width, S * min(width, 40) + 2, 32, lens, 1, layers=1)
    for _ in range(2):
        parents = rng.integers(0, S, S)
        parents[rng.random(S) < 0.1] = -1
        run_reorder(pg, pool, parents)
        assert np.array_equal(counted(pool), pool.refs)


@pytest.mark.parametrize("parents", [[0, 1, 2, 3], [1, 0, 3, 2], [1, 2, 3, 0], [0, 0, 0, 0], [3, 3, 3, 3],
                                     [-1, -1, -1, -1], [2, 2, 9, -5], [1, 1, 0, 0]])
def test_reorder_pages_maps(pg, parents):
    rng = np.random.default_rng(1)
    for lens in ([40, 40, 40, 40], [32, 64, 33, 0]):
        run_reorder(pg, pool_of(rng, 4, 3, 12, 32, lens), parents)


def test_reorder_needs_no_spare_page(pg):
    """Beams of one length in a full pool: those that end give the pages that the
    copies take."""
    rng = np.random.default_rng(2)
    pool = pool_of(rng, 6, 2, 12, 32, [50] * 6)
    assert (pool.refs > 0).all()
    for parents in ([0, 0, 0, 0, 0, 0], [5, 4, 3, 2, 1, 0], [1, 1, 1, 3, 3, 3]):
        assert run_reorder(pg, pool, parents).all()


def test_reorder_without_pages(pg):
    """Sequences of unlike lengths in a full pool: in order, until none is free."""
    rng = np.random.default_rng(2)
    pool = pool_of(rng, 5, 3, 8, 32, [90, 64, 32, 10, 32])
    pool.tables[0, 1] = -1  # evicted
    pool.refs[:] = counted(pool)
    spare = np.flatnonzero(pool.refs == 0)
    pool.tables[2, 1:1 + len(spare)] = spare[:2]  # reserved behind its rows
    pool.refs[:] = counted(pool)
    want = run_reorder(pg, pool, [0, 0, 0, 3, 3])
    assert want.tolist()[0] == 1


def test_reorder_in_a_graph(pg):
    rng = np.random.default_rng(11)
    S, page = 8, 32
    pool = pool_of(rng, S, 4, 40, page, [70] * S, 1)
    pages = [dev(p) for p in pool.pages]
    t, r, n = dev(pool.tables), dev(pool.refs), dev(pool.lengths)
    par = ints(np.arange(S))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        pg.kv_pages_reorder(pages, t, r, n, par)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        granted = pg.kv_pages_reorder(pages, t, r, n, par)
    for _ in range(4):
        parents = rng.integers(0, S, S)
        par.copy_(ints(parents))
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(granted), OB.reorder(pool, parents))
        assert np.array_equal(host(t), pool.tables) and np.array_equal(host(r), pool.refs)
        for a, b in zip(pages, pool.pages):
            assert np.array_equal(host(a), b)


# ---------------------------------------------------------------------------
# reordering contiguous caches
# ---------------------------------------------------------------------------

def cache_of(rng, B, Hkv, cap, D, sb):
    lead = (B, Hkv, cap)
    return [rng.integers(0, 2**32, lead + (D // 8,), dtype=np.uint32) if i % 3 == 0
            else rng.standard_normal(lead + (D // 64,)).astype(sb) for i in range(6)]


@pytest.mark.parametrize("sb", [np.float16, np.float32])
@pytest.mark.parametrize("B,Hkv,cap,D", [(1, 1, 5, 64), (2, 3, 33, 64), (4, 2, 130, 128), (7, 1, 65, 192),
                                         (16, 2, 300, 256), (5, 1, 40, 512), (33, 1, 1000, 64), (1024, 1, 9, 64)])
def test_reorder_cache(gpu, B, Hkv, cap, D, sb):
    rng = np.random.default_rng(B + cap)
    old = cache_of(rng, B, Hkv, cap, D, sb)
    lens = rng.integers(0, cap + 1, B).astype(np.int32)
    lens[0] = cap + 7  # a ring that has gone round
    maps = [np.arange(B), np.roll(np.arange(B), 1), np.arange(B)[::-1], np.zeros(B, int), rng.integers(0, B, B),
            rng.permutation(B), np.where(rng.random(B) < 0.4, -1, rng.integers(0, B, B)), np.full(B, B)]
    t, n = [dev(x) for x in old], dev(lens)
    for parents in maps:
        gpu.kv_reorder_int4(*t, n, ints(parents))
        old, lens = OB.reorder_rows(old, lens, parents)
        assert np.array_equal(host(n), lens)
        for a, b in zip(t, old):
            assert np.array_equal(host(a), b)


@pytest.mark.parametrize("B", [63, 64, 65])
def test_reorder_cache_of_a_waves_sequences(gpu, B):
    """Both sizes of the plan: a ring of all sequences, one parent of all, and none."""
    from gemma4metal_amd import turboquant as tq
    rng = np.random.default_rng(B)
    Hkv, cap, D = 1, 37, 64
    lens = rng.integers(0, cap + 1, B).astype(np.int32)
    x = [rng.integers(0, 2**32, (B, Hkv, cap, D // 8), dtype=np.uint32) if i % 3 == 0
         else rng.standard_normal((B, Hkv, cap, D // 64)).astype(np.float16) for i in range(6)]
    for parents in (np.roll(np.arange(B), 1), np.full(B, B - 1), np.full(B, -1), np.arange(B) // 2):
        d, n = [dev(t) for t in x], dev(lens)
        tq.kv_reorder_int4(*d, n, ints(parents))
        par = np.where((parents >= 0) & (parents < B), parents, -1)
        assert np.array_equal(host(n), np.where(par >= 0, lens[par], 0))
        for t, got in zip(x, d):
            want = t.copy()
            for b in range(B):
                if par[b] >= 0:
                    want[b, :, :lens[par[b]]] = t[par[b], :, :lens[par[b]]]
            assert np.array_equal(host(got), want)


def test_reorder_cache_class_and_graph(gpu):
    rng = np.random.default_rng(1)
    c = gpu.Int4KVCache(4, 2, 40, 128, "cuda", ring=True)
    k, v = (queries(rng, (4, 2, 50, 128), "bf16")[0] for _ in range(2))
    c.append(k, v)
    old, lens = [host(x) for x in c.tensors()], host(c.lengths)
    par = ints([0, 1, 2, 3])
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        c.reorder(par)
    for parents in ([1, 0, 0, 2], [2, 2, 3, 1], [0, 0, 0, 0]):
        par.copy_(ints(parents))
        g.replay()
        torch.cuda.synchronize()
        old, lens = OB.reorder_rows(old, lens, parents)
        assert np.array_equal(host(c.lengths), lens)
        for a, b in zip(c.tensors(), old):
            assert np.array_equal(host(a), b)
    with pytest.raises(ValueError, match="parents"):
        c.reorder(ints([0, 1]))


# ---------------------------------------------------------------------------
# a search
# ---------------------------------------------------------------------------

class Toy:
    """A layer with a vocabulary: rows and logits of a token, on both sides alike."""

    def __init__(self, V, Hkv, Hq, D):
        rng = np.random.default_rng(77)
        bf = lambda *s: O.bf16_bits_to_f32(O.f32_to_bf16_bits(rng.standard_normal(s).astype(np.float32)))  # noqa: E731
        self.k, self.v, self.q = bf(V, Hkv, D), bf(V, Hkv, D), bf(V, Hq, D) * np.float32(0.125)
        self.out = (bf(Hq * D, V) * np.float32(0.125)).astype(np.float32)


@pytest.mark.parametrize("paged", [True, False])
def test_a_search_with_a_cache(gpu, bm, pg, paged):
    """Two requests with three beams each: every step's beams, and the cache behind
    them, as if each beam's tokens had been appended alone."""
    V, Hkv, Hq, D, W, G, page, steps = 50, 2, 4, 128, 3, 2, 32, 7
    toy, S = Toy(V, Hkv, Hq, D), G * W
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, V, (G, 62))
    bf = lambda a: torch.from_numpy(a).cuda().to(torch.bfloat16)  # noqa: E731
    if paged:
        c = pg.PagedInt4KVCache(S * 3, page, S, 4, Hkv, D, "cuda")
    else:
        c = gpu.Int4KVCache(S, Hkv, 80, D, "cuda")
    seqs = [list(prompt[g]) for g in range(G) for _ in range(W)]
    toks = np.array(seqs)
    rows = lambda t: (bf(toy.k[t].transpose(0, 2, 1, 3)), bf(toy.v[t].transpose(0, 2, 1, 3)))  # noqa: E731
    if paged:
        n = ints([62] * S)
        assert host(c.reserve(n)).all()
        c.append(0, *(x.contiguous() for x in rows(toks)))
        c.advance(n)
    else:
        c.append(*(x.contiguous() for x in rows(toks)))
    scores = torch.tensor([[0.0] + [-np.inf] * (W - 1)] * G, device="cuda")
    last = toks[:, -1]
    one = ints([1] * S)
    for _ in range(steps):
        q = bf(toy.q[last])
        o = c.attend(0, q, 2, new=0) if paged else c.attend(q, 2)
        x = o.flatten(1) @ torch.from_numpy(toy.out).cuda()
        old = host(scores)
        val, parents, tokens = OB.beam_select(x.float().cpu().numpy().reshape(G, W, V), old, W)
        scores, par, tok = bm.beam_step(c, x.reshape(G, W, V), scores)
        assert np.array_equal(host(par), parents) and np.array_equal(host(tok), tokens)
        seqs = [seqs[p] + [t] for p, t in zip(parents.ravel(), tokens.ravel())]
        last = tokens.ravel()
        new = rows(last[:, None])
        if paged:
            assert host(c.reserve(one)).all()
            c.append(0, *(y.contiguous() for y in new))
            assert host(c.advance(one)).all()
        else:
            c.append(*(y.contiguous() for y in new))
    # the cache of each beam: its own tokens' rows
    L = len(seqs[0])
    fresh = gpu.Int4KVCache(S, Hkv, L, D, "cuda")
    fresh.append(*(x.contiguous() for x in rows(np.array(seqs))))
    for a, b in zip(c.tensors(), fresh.tensors()):
        a, b = host(a), host(b)
        for s in range(S):
            if paged:
                t = host(c.block_tables)[s]
                mine = np.concatenate([a[0, t[e]] for e in range(-(-L // page))], 1)[:, :L]
            else:
                mine = a[s, :, :L]
            assert np.array_equal(mine, b[s])
    assert len({tuple(s) for s in seqs[:W]}) == W and len({tuple(s) for s in seqs[W:]}) == W


def test_other_device_or_stream_arguments(bm, pg):
    x = torch.zeros(1, 2, 8, device="cuda")
    sc = torch.zeros(1, 2, device="cuda")
    for bad, word in ((dict(scores=sc[0]), "scores"), (dict(scores=sc.double()), "scores"),
                      (dict(finished=sc), "finished"), (dict(logits=x[0]), "logits"), (dict(logits=x.int()), "logits"),
                      (dict(logits=x.transpose(1, 2)), "vocabulary|scores"), (dict(num_out=0), "num_out"),
                      (dict(scores=sc.cpu()), "scores"), (dict(workspace=torch.zeros(1, dtype=torch.uint8, device="cuda")), "workspace")):
        args = dict(logits=x, scores=sc) | bad
        with pytest.raises(ValueError, match=word):
            bm.beam_select(**args)
    from gemma4metal_amd._lib import TQError
    for bad, word in ((dict(num_out=65), "num_out"), (dict(pad_token=8), "pad_token"), (dict(pad_token=-1), "pad_token")):
        with pytest.raises(TQError, match=word):
            bm.beam_select(x, sc, **bad)


def test_a_step_is_refused_before_any_cache_moves(gpu, bm):
    a, b = gpu.Int4KVCache(2, 1, 8, 128, "cuda"), gpu.Int4KVCache(3, 1, 8, 128, "cuda")
    a.lengths.copy_(ints([5, 3]))
    x = torch.zeros(1, 2, 8, device="cuda")
    x[0, 1, 3] = 9.0
    with pytest.raises(ValueError, match="every cache"):
        bm.beam_step([a, b], x, torch.zeros(1, 2, device="cuda"))
    assert host(a.lengths).tolist() == [5, 3]
    parents = bm.beam_step((a,), x, torch.zeros(1, 2, device="cuda"))[1]
    assert host(parents)[0, 0] == 1 and host(a.lengths)[0] == 3
