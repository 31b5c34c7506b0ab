"""GPU: steps of a beam search over several caches: layers with one lengths tensor, caches
that are not fit for it, and beams that find no page."""
import numpy as np
import pytest
import torch

from oracle import beam as OB
from tests.gpu_util import dev, host
from tests.test_gpu_beam import cache_of, ints

pytestmark = pytest.mark.gpu


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


def choice(parents, V=40):
    """Logits and scores of one request whose next beams are these parents'."""
    W = len(parents)
    x = np.zeros((1, W, V), np.float32)
    for k, w in enumerate(parents):
        x[0, w, 3 * k] = 30.0 - 2 * k
    taken = sorted(set(parents))
    scores = np.full((1, W), -np.inf, np.float32)
    for w in taken:  # a beam's total: its score and its logit, less about its largest
        scores[0, w] = max(30.0 - 2 * k for k in range(W) if parents[k] == w)
    return dev(x), dev(scores)


def layers(gpu, rng, B, cap, count, share):
    caches, old = [], []
    for i in range(count):
        c = gpu.Int4KVCache(B, 2, cap, 64, "cuda")
        old.append(cache_of(rng, B, 2, cap, 64, np.float16))
        for t, x in zip(c.tensors(), old[-1]):
            t.copy_(dev(x))
        if share and i:
            c.lengths = caches[0].lengths
        caches.append(c)
    return caches, old


@pytest.mark.parametrize("parents", [[1, -1, 2], [2, 2, 0], [1, 2, 0]])
def test_layers_with_one_lengths_tensor(gpu, parents):
    """Every layer moves the rows of the lengths before the step; the last call sets them."""
    rng = np.random.default_rng(3)
    lens = np.array([3, 17, 9], np.int32)
    caches, old = layers(gpu, rng, 3, 20, 3, True)
    caches[0].lengths.copy_(dev(lens))
    for i, c in enumerate(caches):
        c.reorder(ints(parents), set_lengths=i == len(caches) - 1)
    for c, x in zip(caches, old):
        want, n = OB.reorder_rows(x, lens, parents)
        assert np.array_equal(host(c.lengths), n)
        for a, b in zip(c.tensors(), want):
            assert np.array_equal(host(a), b)
    n = dev(lens)
    gpu.kv_reorder_int4(*caches[0].tensors(), n, ints(parents), set_lengths=False)
    assert np.array_equal(host(n), lens)


@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("parents", [[1, 1, 2], [2, 0, 0], [0, 2, 1]])
def test_a_step_of_several_layers(gpu, bm, parents, share):
    rng = np.random.default_rng(5)
    lens = np.array([2, 19, 8], np.int32)
    caches, old = layers(gpu, rng, 3, 20, 3, share)
    for c in caches:
        c.lengths.copy_(dev(lens))
    x, scores = choice(parents)
    got = bm.beam_step(caches, x, scores)
    assert host(got[1]).tolist() == [parents]
    for c, y in zip(caches, old):
        want, n = OB.reorder_rows(y, lens, parents)
        assert np.array_equal(host(c.lengths), n)
        for a, b in zip(c.tensors(), want):
            assert np.array_equal(host(a), b)


def test_caches_that_a_step_cannot_move(gpu, bm, pg):
    """A cache twice, lengths that overlap or are not int32, pages that share their
    lengths or their tables: refused before anything moves."""
    x, scores = choice([1, 1])
    make = lambda: gpu.Int4KVCache(2, 1, 8, 64, "cuda")  # noqa: E731
    pool = lambda: pg.PagedInt4KVCache(4, 32, 2, 2, 1, 64, "cuda")  # noqa: E731
    a = make()
    a.lengths.copy_(ints([5, 3]))

    def refused(other, word):
        with pytest.raises(ValueError, match=word):
            bm.beam_step([a, other], x, scores)
        assert host(a.lengths).tolist() == [5, 3]
    refused(a, "twice")
    b = make()
    b.kq = a.kq
    refused(b, "twice")
    long = torch.zeros(3, dtype=torch.int32, device="cuda")
    keep, a.lengths = a.lengths, long[:2]
    a.lengths.copy_(keep)
    b = make()
    b.lengths = long[1:]
    refused(b, "lengths")
    a.lengths = keep
    b.lengths = keep.long()
    refused(b, "lengths")
    b.lengths = torch.zeros(4, dtype=torch.int32, device="cuda")[::2]
    refused(b, "lengths")
    p = pool()
    p.lengths = a.lengths
    refused(p, "lengths")
    p, r = pool(), pool()
    r.block_tables = p.block_tables
    with pytest.raises(ValueError, match="tables|twice"):
        bm.beam_step([p, r], x, scores)


def test_a_beam_without_a_page_has_no_score(gpu, bm, pg):
    """A request's first step in a full pool: one beam goes on, the other finds no page
    for its copy of the last one.  It is no beam of the next step either."""
    rng = np.random.default_rng(9)
    c = pg.PagedInt4KVCache(2, 32, 2, 2, 1, 64, "cuda")
    other = gpu.Int4KVCache(2, 1, 64, 64, "cuda")
    n = ints([40, 0])
    assert host(c.reserve(n)).tolist() == [1, 0]
    k = torch.from_numpy(rng.standard_normal((2, 1, 40, 64)).astype(np.float32)).cuda()
    c.append(0, k, k)
    c.advance(n)
    other.append(k, k, advance=False)
    other.lengths.copy_(c.lengths)
    x, scores = choice([0, 0])
    for caches in ([c, other], [c]):
        got = bm.beam_step(caches, x, scores)
        assert host(got[1]).tolist() == [[0, 0]]
        assert host(c.lengths).tolist() == [40, 0]
        s = host(got[0])
        assert np.isfinite(s[0, 0]) and s[0, 1] == -np.inf
    x, _ = choice([0, 1])
    assert host(bm.beam_step(c, x, got[0])[1]).tolist() == [[0, 0]]  # both of the one that is left


def test_numbers_past_32_bits(bm, pg):
    """They are refused, not cut off to others."""
    x, scores = choice([0, 1])
    for name in ("pad_token", "num_out"):
        with pytest.raises(ValueError, match=name):
            bm.beam_select(x, scores, **{name: 2**32 + 1})
    pages = [torch.zeros((2, 1, 32, n), dtype=t, device="cuda") for n, t in
             ((16, torch.uint32), (2, torch.float16), (2, torch.float16)) * 2]
    q = torch.zeros((2, 1, 128), device="cuda")
    t, st, n = ints([[0], [1]]), ints([0, 1, 2]), ints([5, 7])
    ok = dict(gqa_factor=1, sliding_window=0, num_sinks=0, max_new=1, max_kv_len=32)
    pg.sdpa_int4_paged_chunks(q, *pages, t, st, n, **ok)
    for name, value in ok.items():
        with pytest.raises(ValueError, match=name):
            pg.sdpa_int4_paged_chunks(q, *pages, t, st, n, **(ok | {name: 2**32 + value}))
