"""GPU: attention of a chunk of new tokens of every sequence of a batch over its pages,
against the oracle in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import paged as OP
from tests.gpu_util import dev, host, queries
from tests.test_gpu_paged import close, ints, make_pool, random_tables, spoil
from tests.test_gpu_paged_calls import TILES, definition, within

pytestmark = pytest.mark.gpu

SHAPES = [(2, 1, 128, 32), (16, 4, 128, 64), (4, 2, 256, 64), (8, 1, 256, 32), (4, 2, 512, 32), (8, 1, 512, 64), (3, 1, 128, 128)]


@pytest.fixture(scope="module")
def pg():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from gemma4metal_amd import paged
    return paged


def batch(rng, new, lens, Hq, Hkv, D, page, sb="f16", qt="bf16", spare=0):
    """Queries, pages (NaN where no sequence has rows), tables and starts."""
    N = sum(-(-max(n, 0) // page) for n in lens) + 1
    width = max(max(-(-n // page) for n in lens), 1) + spare
    tables = random_tables(rng, lens, page, N, width)
    pages = make_pool(rng, N, Hkv, page, D, sb)
    spoil(pages, tables, lens, page)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q, qf = queries(rng, (int(starts[-1]), Hq, D), qt)
    return q, qf, pages, tables, starts


def run(pg, q, pages, tables, starts, lens, gqa, *a, **kw):
    return host(pg.sdpa_int4_paged_chunks(q, *[dev(p) for p in pages], dev(tables), ints(starts), ints(lens), gqa, *a, **kw))


@pytest.mark.parametrize("Hq,Hkv,D,page", SHAPES)
@pytest.mark.parametrize("new,prior,window,sinks", [([1], [0], 0, 0), ([3, 1, 0, 17], [0, 30, 5, 64], 0, 0),
                                                    ([70, 1, 33], [31, 200, 0], 50, 0),
                                                    ([2, 65, 5], [300, 97, 1], 100, 4),
                                                    ([5, 5, 5, 5, 5], [900, 1, 63, 64, 400], 64, 70)])
def test_chunks(pg, Hq, Hkv, D, page, new, prior, window, sinks):
    rng = np.random.default_rng(sum(new) + D)
    lens = [n + m for n, m in zip(new, prior)]
    q, qf, pages, tables, starts = batch(rng, new, lens, Hq, Hkv, D, page)
    ref = OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, page, Hq // Hkv, 1.0, window, sinks)
    for kw in ({}, dict(max_new=max(new)), dict(max_kv_len=max(lens), max_new=max(new))):
        close(run(pg, q, pages, tables, starts, lens, Hq // Hkv, 1.0, window, sinks, **kw), ref, str(kw))


@pytest.mark.parametrize("sb,qt", [("f16", "f16"), ("f32", "f32"), ("f16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 2, 256), (8, 1, 512)])
def test_types_and_many_rows(pg, Hq, Hkv, D, sb, qt):
    """Blocks of 64 and of 128 rows, some of them split."""
    rng = np.random.default_rng(D)
    new, lens = [40, 150, 1], [2100, 150, 700]
    q, qf, pages, tables, starts = batch(rng, new, lens, Hq, Hkv, D, 64, sb, qt)
    ref = OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, 64, Hq // Hkv, 0.3)
    for most in (None, 150):
        close(run(pg, q, pages, tables, starts, lens, Hq // Hkv, 0.3, max_new=most, max_kv_len=2100), ref)


@pytest.mark.parametrize("sb,qt", [("f16", "bf16"), ("f32", "f32"), ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("Hq,Hkv,D", [(6, 3, 128), (12, 3, 256), (8, 1, 512)])
@pytest.mark.parametrize("new,prior,window,sinks", [([1, 70, 3, 1, 2, 90, 1], [900, 10, 2100, 0, 33, 700, 64], 0, 0),
                                                    ([129, 1, 0, 1], [0, 5, 9, 2600], 300, 4),
                                                    ([1, 65], [3000, 0], 0, 0), ([64, 1, 64], [40, 1, 3000], 0, 0)])
def test_long_chunks_and_few_rows_in_one_call(pg, Hq, Hkv, D, sb, qt, new, prior, window, sinks):
    """Jobs of both kinds, odd numbers of either, split and whole; again after a call
    that left other partials, bit by bit."""
    rng = np.random.default_rng(len(new) + D)
    lens = [n + m for n, m in zip(new, prior)]
    q, qf, pages, tables, starts = batch(rng, new, lens, Hq, Hkv, D, 64, sb, qt)
    ref = OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, 64, Hq // Hkv, 0.4, window, sinks)
    kw = dict(max_new=max(new), max_kv_len=max(lens))
    got = run(pg, q, pages, tables, starts, lens, Hq // Hkv, 0.4, window, sinks, **kw)
    close(got, ref)
    run(pg, q, pages, tables, starts, lens, Hq // Hkv, 3.0)
    assert np.array_equal(got, run(pg, q, pages, tables, starts, lens, Hq // Hkv, 0.4, window, sinks, **kw))


@pytest.mark.parametrize("B", [63, 64, 65, 200])
def test_more_sequences_than_a_wave(pg, B):
    rng = np.random.default_rng(B)
    new = rng.integers(0, 4, B).tolist()
    new[-1], new[0] = 9, 2
    lens = [n + int(x) for n, x in zip(new, rng.integers(0, 90, B))]
    lens[-1] += 1500
    q, qf, pages, tables, starts = batch(rng, new, lens, 4, 2, 128, 32)
    ref = OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, 32, 2)
    close(run(pg, q, pages, tables, starts, lens, 2), ref)


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 128), (4, 2, 256), (8, 1, 512)])
def test_precision(pg, Hq, Hkv, D):
    rng = np.random.default_rng(D + 1)
    new, lens, page = [70, 6], [1777, 900], 64
    for sb, qt in (("f16", "bf16"), ("f32", "f32")):
        q, qf, pages, tables, starts = batch(rng, new, lens, Hq, Hkv, D, page, sb, qt)
        got = run(pg, q, pages, tables, starts, lens, Hq // Hkv, D**-0.5)
        for b, L in enumerate(lens):
            mine = slice(starts[b], starts[b + 1])
            ref = definition(qf[mine], pages, tables[b], range(L - new[b] + 1, L + 1), page, Hq // Hkv, D**-0.5)
            within(got[mine], ref, TILES, f"sequence {b}")


def test_missing_pages_short_lengths_and_rows_behind(pg):
    """Entries without a page, lengths below the chunk or below 0, lengths past
    max_kv_len, and rows behind the last chunk, which stay."""
    rng = np.random.default_rng(3)
    Hq, Hkv, D, page = 4, 2, 256, 32
    new, lens = [4, 3, 5, 2, 6], [200, 120, 90, 64, 300]
    q, qf, pages, tables, starts = batch(rng, new, lens, Hq, Hkv, D, page)
    tables[0, 1], tables[0, 2], tables[1, :], tables[2, 2] = -1, 10**6, -1, -1
    lens[3], lens[2] = 1, -7   # the first of two queries stands before the sequence
    q, qf = queries(rng, (int(starts[-1]) + 3, Hq, D), "bf16")
    ref = OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, page, 2, 1.0, 0, 0, 256)
    assert not ref[starts[1]:starts[3]].any() and not ref[starts[3]].any() and ref[starts[3] + 1].any()
    out = torch.full((q.shape[0], Hq, D), 7.0, device="cuda")
    got = run(pg, q, pages, tables, starts, lens, 2, max_kv_len=256, out=out)
    close(got[:starts[-1]], ref[:starts[-1]])
    assert (got[starts[-1]:] == 7).all()
    # a batch without tokens, and one without queries
    assert (run(pg, q, pages, tables, [0] * 6, lens, 2, out=out.fill_(3.0)) == 3).all()
    assert run(pg, q[:0], pages, tables, [0] * 6, lens, 2).shape == (0, Hq, D)


@pytest.mark.parametrize("big", [1e-30, 1e25, 1e36])
@pytest.mark.parametrize("D,new", [(128, 3), (256, 3), (256, 60), (512, 1), (512, 30)])
def test_any_range_of_v_scales(pg, D, new, big):
    """V scales and biases of fp32 caches near the ends of fp32, one key far above the
    others (some rows attend it, some do not), and groups far apart."""
    rng = np.random.default_rng(D)
    Hq, Hkv, page, lens = 4, 2, 32, [new + 70, new]
    q, qf, pages, tables, starts = batch(rng, [new, new], lens, Hq, Hkv, D, page, "f32", "f32")
    for i in (4, 5):
        pages[i] *= np.float32(big)
        pages[i][..., 0] *= np.float32(1e-7)
    for t in (40, lens[0] - 1):          # keys of sequence 0
        e = tables[0, t // page]
        for i in (4, 5):
            pages[i][e, :, t % page] *= np.float32(100)
    ref = OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, page, 2, 0.05)
    got = run(pg, q, pages, tables, starts, lens, 2, 0.05).astype(np.float64)
    # By group of 64 dims: a group's precision is its own.  Weights are at most 2^8 and are
    # summed before they are divided by their sum: values of more than 2^128 / (2^8 keys)
    # may overflow (at 1e36 all do, and infinities come of times 100), to infinity or NaN.
    most = np.abs(pages[4]).max(axis=(0, 1, 2)) * 15 + np.abs(pages[5]).max(axis=(0, 1, 2))
    for g in range(D // 64):
        a, b = got[..., 64 * g:64 * g + 64], ref[..., 64 * g:64 * g + 64]
        fine = np.isfinite(a).all(-1)
        assert fine.all() or not most[g] < 2.0**128 / (2.0**8 * lens[0]), g
        a, b = a[fine] / big, b[fine] / big
        err = np.linalg.norm(a - b, axis=-1) / np.linalg.norm(b, axis=-1)
        assert fine.sum() == 0 or err.max() <= 1e-4, (g, err.max())


def test_infinite_values_stay_with_who_attends_them(pg):
    """A key with infinite V scales or biases, or NaN ones: only the queries that see it
    have them in their results."""
    rng = np.random.default_rng(8)
    for D, new in ((128, 5), (256, 60), (512, 2), (512, 30)):
        Hq, Hkv, page, lens = 4, 2, 32, [new + 100]
        q, qf, pages, tables, starts = batch(rng, [new], lens, Hq, Hkv, D, page)
        t = lens[0] - 1                   # the last query's own key
        for i, bad in ((4, np.inf), (5, np.nan), (1, np.nan)):
            p = [x.copy() for x in pages]
            p[i][tables[0, t // page], :, t % page] = bad
            got = run(pg, q, p, tables, starts, lens, 2)
            with np.errstate(invalid="ignore"):
                ref = OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, page, 2)
            close(got[:-1], ref[:-1])
            assert not np.isfinite(got[-1]).all()


def test_starts_that_do_not_ascend(pg):
    """Nothing can be said of the result, but nothing else is touched either."""
    rng = np.random.default_rng(12)
    new, lens = [2, 3, 1], [700, 900, 300]
    q, qf, pages, tables, starts = batch(rng, new, lens, 4, 2, 128, 32)
    d, t, n = [dev(p) for p in pages], dev(tables), ints(lens)
    ws = torch.zeros(1 << 26, dtype=torch.uint8, device="cuda")
    big = torch.full((40, 4, 128), 5.0, device="cuda")
    call = lambda st: pg.sdpa_int4_paged_chunks(q, *d, t, ints(st), n, 2, out=big[16:22], max_kv_len=900, workspace=ws)  # noqa: E731
    need = pg._chunks_ws_size(3, 6, 4, 2, 128, 6, 900)
    ws[need:] = 77
    for bad in ([0, 6, 0, 6], [6, 0, 6, 0], [-9, 100, -9, 100], [2**31 - 1, -2**31, 2**31 - 1, 5]):
        call(bad)
        torch.cuda.synchronize()
        assert (big[:16] == 5).all() and (big[22:] == 5).all() and (ws[need:] == 77).all() and not ws[:1 << 18].any()
    close(host(call(starts)), OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, 32, 2))


def test_equal_to_the_calls_it_stands_for(pg):
    """A prompt's chunks one after the other, and single tokens, as the calls of one
    sequence and of one token have them."""
    rng = np.random.default_rng(4)
    Hq, Hkv, D, page = 8, 2, 128, 32
    lens = [333, 1, 64, 500]
    q, qf, pages, tables, starts = batch(rng, [1] * 4, lens, Hq, Hkv, D, page)
    d = [dev(p) for p in pages]
    one = host(pg.sdpa_int4_paged(q, *d, dev(tables), ints(lens), 4, 1.0, 100, 5))
    close(run(pg, q, pages, tables, starts, lens, 4, 1.0, 100, 5), one.astype(np.float64))
    q, _ = queries(rng, (170, Hq, D), "bf16")
    whole = host(pg.sdpa_int4_paged_prefill(q, *d, dev(tables[3]), 330, 4, 1.0, 100, 5))
    got = [run(pg, q[a:z].contiguous(), pages, tables[3:], [0, z - a], [330 + z], 4, 1.0, 100, 5)
           for a, z in ((0, 64), (64, 65), (65, 170))]
    close(np.concatenate(got), whole.astype(np.float64))


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 256), (8, 1, 512)])
def test_one_graph_for_all_lengths(pg, Hq, Hkv, D):
    rng = np.random.default_rng(6)
    B, N, page, width = 5, 60, 32, 40
    lens = [1000, 40, 33, 500, 64]
    tables = random_tables(rng, [width * page] * B, page, B * width, width)
    pages = make_pool(rng, B * width, Hkv, page, D, "f16")
    d, t, n, st = [dev(p) for p in pages], dev(tables), ints(lens), ints([0, 1, 2, 3, 4, 5])
    q, qf = queries(rng, (N, Hq, D), "bf16")
    s = torch.cuda.Stream()
    call = lambda: pg.sdpa_int4_paged_chunks(q, *d, t, st, n, Hq // Hkv, 0.5, max_kv_len=1280)  # noqa: E731
    with torch.cuda.stream(s):
        call()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        got = call()
    for new, lens in (([1] * 5, [1000, 40, 33, 500, 64]), ([40, 0, 2, 1, 17], [1280, 9, 2, 1, 200]),
                      ([0, 0, 60, 0, 0], [5, 5, 700, 5, 5])):
        starts = np.concatenate([[0], np.cumsum(new)])
        st.copy_(ints(starts))
        n.copy_(ints(lens))
        g.replay()
        torch.cuda.synchronize()
        ref = OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, page, Hq // Hkv, 0.5)
        close(host(got)[:starts[-1]], ref[:starts[-1]])
        with torch.cuda.stream(s):
            eager = call()
        s.synchronize()
        assert torch.equal(eager[:starts[-1]], got[:starts[-1]])


def test_a_serving_run_with_chunks(pg):
    """Prompts in parts beside sequences that go on, as one call a step, and decode
    calls in between with the same workspace."""
    rng = np.random.default_rng(9)
    Hq, Hkv, D, page, S = 4, 2, 128, 32, 3
    c = pg.PagedInt4KVCache(20, page, S, 6, Hkv, D, "cuda")
    pool = OP.Pool(np.full((S, 6), -1, np.int32), np.zeros(20, np.int32), np.zeros(S, np.int32), page,
                   [host(t) for t in c.tensors()])
    for n in ([50, 0, 0], [1, 40, 0], [1, 23, 7], [1, 1, 60], [4, 1, 5]):
        assert host(c.reserve(ints(n))).tolist() == pool.reserve(n).tolist()
        parts = []
        for s in range(S):
            (k, kf), (v, vf) = queries(rng, (Hkv, n[s], D), "bf16"), queries(rng, (Hkv, n[s], D), "bf16")
            if n[s]:
                c.append_one(0, s, k, v)
                OP.append([p[0] for p in pool.pages], kf[None], vf[None], pool.tables[s:s + 1], pool.lengths[s:s + 1],
                          page, "f16")
            parts.append(n[s])
        starts = np.concatenate([[0], np.cumsum(parts)]).astype(np.int32)
        q, qf = queries(rng, (int(starts[-1]), Hq, D), "bf16")
        lens = pool.lengths + np.array(n)
        got = c.attend_chunks(0, q, ints(starts), 2, 1.0, 48, 3)
        close(host(got), OP.sdpa_int4_paged_chunks(qf, [p[0] for p in pool.pages], pool.tables, starts, lens, page, 2, 1.0, 48, 3))
        assert host(c.advance(ints(n))).tolist() == pool.advance(n).tolist()
        q, qf = queries(rng, (S, Hq, D), "bf16")
        close(host(c.attend(0, q, 2, new=0)), OP.sdpa_int4_paged(qf, [p[0] for p in pool.pages], pool.tables, pool.lengths, page, 2))


def test_refusals(pg):
    from gemma4metal_amd._lib import TQError
    rng = np.random.default_rng(1)
    q, _, pages, tables, starts = batch(rng, [2, 1], [40, 9], 4, 2, 128, 32)
    d, t, st, n = [dev(p) for p in pages], dev(tables), ints(starts), ints([40, 9])
    ok = lambda **kw: pg.sdpa_int4_paged_chunks(kw.pop("q", q), *kw.pop("pages", d), kw.pop("t", t), kw.pop("st", st),  # noqa: E731
                                                kw.pop("n", n), kw.pop("gqa", 2), **kw)
    ok()
    for bad, word in ((dict(st=ints([0, 2])), "starts"), (dict(st=st.long()), "starts"), (dict(n=n[:1]), "seq_lens"),
                      (dict(t=t[0]), "block_tables"), (dict(q=q[0]), "queries"), (dict(q=q.cpu()), "queries"),
                      (dict(st=st.cpu()), "starts"), (dict(out=torch.empty(3, 4, 64, device="cuda")), "out"),
                      (dict(pages=d[:5] + d[:1]), "v_biases")):
        with pytest.raises(ValueError, match=word):
            ok(**bad)
    for bad, word in ((dict(gqa=1), "num_heads"), (dict(max_kv_len=10**6), "max_kv_len"), (dict(max_kv_len=-1), "max_kv_len"),
                      (dict(max_new=-1), "max_new"), (dict(sliding_window=-1), "sliding_window"),
                      (dict(num_sinks=-1), "num_sinks"), (dict(scale=float("nan")), "scale")):
        with pytest.raises(TQError, match=word):
            ok(**bad)
    big = ints([0, 2, 3])
    with pytest.raises(ValueError, match="workspace"):
        wide = torch.full((2, 64), -1, dtype=torch.int32, device="cuda")
        ok(t=wide, st=big, workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    c = pg.PagedInt4KVCache(4, 32, 2, 2, 2, 128, "cuda")
    for bad in (ints([0, 3]), st.long(), st.cpu()):
        with pytest.raises(ValueError, match="starts"):
            c.attend_chunks(0, q, bad, 2)
    assert not host(c.attend_chunks(0, q, ints([0, 0, 0]), 2, out=torch.zeros(3, 4, 128, device="cuda"))).any()
