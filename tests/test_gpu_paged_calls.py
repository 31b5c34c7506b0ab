"""GPU: the paged int4 cache where a step is refused, a batch's prefix is given up
by a sequence, requests are too large, V scales are unlike, and to the precision
that each form states."""
import numpy as np
import pytest
import torch

from oracle import oracle as O
from oracle import paged as OP
from tests.gpu_util import dev, host, queries
from tests.test_gpu_paged import close, ints, make_pool, random_tables, spoil

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pg():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from gemma4metal_amd import paged
    return paged


# ---------------------------------------------------------------------------
# steps that are refused
# ---------------------------------------------------------------------------

def test_a_refused_sequence_is_not_advanced(pg):
    """A sequence without a page for its row keeps its length.  Were it counted, the
    next page it gets would put its last owner's row into the sequence."""
    rng = np.random.default_rng(5)
    Hq, Hkv, D, page = 4, 2, 128, 32
    c = pg.PagedInt4KVCache(4, page, 2, 4, Hkv, D, "cuda")
    pool = OP.Pool(np.full((2, 4), -1, np.int32), np.zeros(4, np.int32), np.zeros(2, np.int32), page,
                   [host(t) for t in c.tensors()])

    def step(n, want):
        """n[s] rows to every sequence; the attention of those that got theirs."""
        ok = host(c.reserve(ints(n)))
        assert ok.tolist() == pool.reserve(n).tolist() == want
        T = max(n)
        (k, kf), (v, vf) = queries(rng, (2, Hkv, T, D), "bf16"), queries(rng, (2, Hkv, T, D), "bf16")
        q, qf = queries(rng, (2, Hq, D), "bf16")
        lens = pool.lengths.copy()
        for s in range(2):
            if n[s]:
                c.append_one(0, s, k[s, :, :n[s]].contiguous(), v[s, :, :n[s]].contiguous())
                OP.append([p[0] for p in pool.pages], kf[s:s + 1, :, :n[s]], vf[s:s + 1, :, :n[s]],
                          pool.tables[s:s + 1], lens[s:s + 1], page, "f16")
        got = c.attend(0, q, 2, 1.0, new=ints(n))
        ref = OP.sdpa_int4_paged(qf, [p[0] for p in pool.pages], pool.tables, lens + np.array(n), page, 2)
        for s in range(2):
            if want[s]:
                close(host(got)[s], ref[s], f"sequence {s}")
        assert host(c.advance(ints(n))).tolist() == pool.advance(n).tolist() == want
        assert np.array_equal(host(c.lengths), pool.lengths)

    step([64, 64], [1, 1])            # all four pages
    step([1, 1], [0, 0])              # both refused: 64 rows stay 64
    assert host(c.lengths).tolist() == [64, 64]
    c.free(ints([0, 1]))
    pool.free([0, 1])
    step([1, 0], [1, 0])              # a page of the sequence that ended: row 64 is the new one
    step([40, 0], [1, 0])
    assert host(c.lengths).tolist() == [105, 0]
    assert host(c.advance(ints([-5, 0]))).tolist() == [0, 0]
    assert host(c.lengths).tolist() == [100, 0]


@pytest.mark.parametrize("S,width,N,page", [(1, 1, 1, 32), (7, 40, 60, 64), (1500, 5, 3000, 32)])
def test_advance_random(pg, S, width, N, page):
    rng = np.random.default_rng(S)
    tables = np.where(rng.random((S, width)) < 0.8, rng.integers(0, N, (S, width)), -1).astype(np.int32)
    tables[rng.random((S, width)) < 0.03] = N
    lens = rng.integers(-2, width * page, S).astype(np.int32)
    ask = np.where(rng.random(S) < 0.8, rng.integers(-3, 3 * page, S), 2**31 - 1).astype(np.int32)
    t, r, n = dev(tables), ints(np.zeros(N)), dev(lens)
    pool = OP.Pool(tables, np.zeros(N, np.int32), lens, page)
    assert np.array_equal(host(pg.kv_pages_advance(t, r, n, dev(ask), page)), pool.advance(ask))
    assert np.array_equal(host(n), pool.lengths) and np.array_equal(host(t), tables)
