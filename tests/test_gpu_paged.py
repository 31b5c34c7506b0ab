"""GPU: the paged int4 cache against its oracle in 64 bits -- append, decode
attention (windows, sinks, shared prefixes), prompts, page operations -- at the
sizes and states where each can go wrong."""
import numpy as np
import pytest
import torch

from oracle import oracle as O
from oracle import paged as OP
from tests.gpu_util import dev, host, queries

pytestmark = pytest.mark.gpu

# Queries are held in 22 bits of fixed point of their row's largest value or as
# two 11-bit parts: at most 2^-22 of it.  With |q| <= 4.5, |k| summed over a
# row <= 0.85 D (RMS-normed), a score is off by 4.5 0.85 512 2^-22 = 5e-4 at the
# very most (D 512; signs in a row: 25 times less), a weight by as much of
# itself, an output by that times |v| <= 5.  Weights add 2^-17.  Its 2-norm
# relative to the result goes by the typical size: 5e-4 / 25 times a few.
ATOL, RTOL = 1e-3, 1e-4


def close(got, ref, what=""):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert got.shape == ref.shape
    assert np.isfinite(got).all(), f"{what}: not finite"
    d = np.abs(got - ref)
    assert d.max() <= ATOL, f"{what}: off by {d.max():.3e}"
    rel = np.linalg.norm(d) / max(np.linalg.norm(ref), 1e-30)
    assert rel <= RTOL, f"{what}: relative {rel:.3e}"


def make_pool(rng, N, Hkv, page, D, sb):
    k = O.quantize_int4(O.rms_norm(rng.standard_normal((N, Hkv, page, D)).astype(np.float32)), sb)
    v = O.quantize_int4(rng.standard_normal((N, Hkv, page, D)).astype(np.float32), sb)
    return list(k) + list(v)


def spoil(pages, tables, lens, page):
    """NaN scales and biases in every row that no sequence has written."""
    used = np.zeros((pages[0].shape[0], page), bool)
    for row, n in zip(tables, lens):
        for t in range(max(int(n), 0)):
            e = row[t // page]
            if 0 <= e < used.shape[0]:
                used[e, t % page] = True
    for i in (1, 2, 4, 5):
        pages[i] = pages[i].copy()
        pages[i][np.broadcast_to(~used[:, None, :, None], pages[i].shape)] = np.nan


def random_tables(rng, lens, page, N, width, shared=0):
    """Tables of distinct pages in any order; the first `shared` entries alike."""
    order = rng.permutation(N).astype(np.int32)
    head, at = order[:shared], shared
    t = np.full((len(lens), width), -1, np.int32)
    for i, n in enumerate(lens):
        t[i, :shared] = head
        k = max(-(-max(int(n), 0) // page) - shared, 0)
        t[i, shared:shared + k] = order[at:at + k]
        at += k
    assert at <= N
    return t


def ints(x):
    return torch.tensor(np.asarray(x, np.int32)).cuda()


@pytest.fixture(scope="module")
def pg():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from gemma4metal_amd import paged
    return paged


SHAPES = [(2, 1, 128), (16, 8, 128), (16, 4, 128), (8, 1, 128), (4, 4, 128), (3, 1, 128), (4, 4, 256), (8, 4, 256),
          (8, 2, 256), (8, 1, 256), (6, 2, 256), (2, 2, 512), (4, 2, 512), (8, 1, 512), (16, 2, 512)]
LENS = [0, 1, 31, 32, 33, 64, 95, 129, 300, 517]


@pytest.mark.parametrize("sb", ["f16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D", SHAPES)
def test_decode_lengths(pg, Hq, Hkv, D, sb):
    rng = np.random.default_rng(Hq * 1000 + D)
    page = {128: 32, 256: 64, 512: 128}[D]
    lens = LENS
    N = sum(-(-n // page) for n in lens) + 2
    tables = random_tables(rng, lens, page, N, -(-max(lens) // page) + 1)
    pages = make_pool(rng, N, Hkv, page, D, sb)
    spoil(pages, tables, lens, page)
    q, qf = queries(rng, (len(lens), Hq, D), {0: "bf16", 1: "f16", 2: "f32"}[(Hq + D // 128 + (sb == "f32")) % 3])
    got = pg.sdpa_int4_paged(q, *map(dev, pages), dev(tables), ints(lens), Hq // Hkv, 0.6)
    ref = OP.sdpa_int4_paged(qf, pages, tables, lens, page, Hq // Hkv, 0.6)
    close(host(got), ref)
    assert not host(got)[0].any()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (31, 4), (64, 33), (100, 64), (100, 97), (40, 400), (2000, 7),
                                          (65, 130)])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 4, 128, 32), (4, 2, 256, 64), (8, 1, 256, 32), (4, 2, 512, 32), (8, 1, 512, 64)])
def test_decode_window_and_sinks(pg, Hq, Hkv, D, page, window, sinks):
    rng = np.random.default_rng(window * 100 + sinks)
    lens = [1, 32, 65, 130, 200, 333, 450]
    N = sum(-(-n // page) for n in lens)
    tables = random_tables(rng, lens, page, N, -(-max(lens) // page))
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    # what lies between the sinks and the window is not read as numbers
    for b, n in enumerate(lens):
        for t in np.flatnonzero(~OP.visible(n, n, window, sinks)):
            for i in (1, 2, 4, 5):
                pages[i][tables[b, t // page], :, t % page] = [np.nan, np.inf][t % 2]
    spoil(pages, tables, lens, page)
    q, qf = queries(rng, (len(lens), Hq, D), "bf16")
    got = pg.sdpa_int4_paged(q, *map(dev, pages), dev(tables), ints(lens), Hq // Hkv, 0.8, window, sinks)
    close(host(got), OP.sdpa_int4_paged(qf, pages, tables, lens, page, Hq // Hkv, 0.8, window, sinks))
    # pages that eviction gives up are not missed
    gone = OP.Pool(tables, np.ones(N), lens, page)
    gone.evict(window, sinks)
    again = pg.sdpa_int4_paged(q, *map(dev, pages), dev(gone.tables), ints(lens), Hq // Hkv, 0.8, window, sinks)
    assert torch.equal(got, again)


def test_decode_windows_per_sequence_and_clamped_lengths(pg):
    rng = np.random.default_rng(8)
    Hq, Hkv, D, page = 4, 2, 256, 32
    lens, wins = [300, 300, 300, -5, 999], [0, 40, 299, 0, 50]
    tables = random_tables(rng, [300, 300, 300, 0, 300], page, 50, 12)
    pages = make_pool(rng, 50, Hkv, page, D, "f16")
    q, qf = queries(rng, (5, Hq, D), "bf16")
    got = pg.sdpa_int4_paged(q, *map(dev, pages), dev(tables), ints(lens), 2, 1.0, 7, 5, windows=ints(wins), max_kv_len=300)
    close(host(got), OP.sdpa_int4_paged(qf, pages, tables, lens, page, 2, 1.0, 7, 5, windows=wins, max_kv_len=300))


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 4, 128), (4, 2, 256), (2, 2, 512), (8, 1, 512)])
def test_decode_bad_pages(pg, Hq, Hkv, D):
    """Entries that name no page take their keys with them, also where nothing
    is left; what the pool's first page holds does not matter."""
    rng = np.random.default_rng(D)
    page, N = 32, 40
    lens = [200, 200, 64, 33, 20, 500]
    tables = random_tables(rng, lens, page, N - 1, 16) + 1
    tables[tables == 0] = -1
    tables[0, 2], tables[1, [0, 5]], tables[2, :2], tables[3, 1], tables[4, 0] = -1, [N, 2**31 - 1], -7, N, -2**31
    tables[5, ::2] = N + 3
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    for i in (1, 2, 4, 5):
        pages[i][0] = np.nan
    q, qf = queries(rng, (len(lens), Hq, D), "f16")
    got = host(pg.sdpa_int4_paged(q, *map(dev, pages), dev(tables), ints(lens), Hq // Hkv, 0.7))
    close(got, OP.sdpa_int4_paged(qf, pages, tables, lens, page, Hq // Hkv, 0.7))
    assert not got[2].any() and not got[4].any()


@pytest.mark.parametrize("Hq,Hkv,D,page,longest", [(8, 4, 256, 64, 6000), (4, 1, 512, 128, 4000), (8, 1, 512, 64, 5000),
                                                   (4, 2, 128, 32, 9000)])
def test_decode_long_sequences(pg, Hq, Hkv, D, page, longest):
    """Splits along the keys and their merge; many sequences of unequal lengths."""
    rng = np.random.default_rng(longest)
    lens = [longest, longest // 3 + 1, 7, longest - 1, 0, 700]
    N = sum(-(-n // page) for n in lens)
    tables = random_tables(rng, lens, page, N, -(-longest // page))
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    spoil(pages, tables, lens, page)
    d = [dev(p) for p in pages]
    q, qf = queries(rng, (len(lens), Hq, D), "bf16")
    for W, sinks in ((0, 0), (1500, 70)):
        ref = OP.sdpa_int4_paged(qf, pages, tables, lens, page, Hq // Hkv, 1.0, W, sinks)
        got = pg.sdpa_int4_paged(q, *d, dev(tables), ints(lens), Hq // Hkv, 1.0, W, sinks)
        close(host(got), ref)
        again = pg.sdpa_int4_paged(q, *d, dev(tables), ints(lens), Hq // Hkv, 1.0, W, sinks)
        assert torch.equal(got, again)
    one = pg.sdpa_int4_paged(q[:1], *d, dev(tables[:1]), ints(lens[:1]), Hq // Hkv, 1.0)
    close(host(one), OP.sdpa_int4_paged(qf[:1], pages, tables[:1], lens[:1], page, Hq // Hkv, 1.0))


def test_decode_more_sequences_than_a_wave(pg):
    rng = np.random.default_rng(70)
    Hq, Hkv, D, page, B = 4, 2, 128, 32, 70
    lens = rng.integers(0, 400, B)
    N = int(sum(-(-n // page) for n in lens))
    tables = random_tables(rng, lens, page, N, 13)
    pages = make_pool(rng, N, Hkv, page, D, "f32")
    q, qf = queries(rng, (B, Hq, D), "f32")
    got = pg.sdpa_int4_paged(q, *map(dev, pages), dev(tables), ints(lens), 2, 1.0, 100, 6)
    close(host(got), OP.sdpa_int4_paged(qf, pages, tables, lens, page, 2, 1.0, 100, 6))


@pytest.mark.parametrize("sb,qt", [("f16", "bf16"), ("f32", "f32"), ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(2, 1, 128, 32), (16, 4, 128, 64), (4, 2, 256, 64), (8, 1, 256, 32),
                                           (6, 2, 256, 128), (4, 2, 512, 32), (8, 1, 512, 128)])
def test_shared_prefix(pg, Hq, Hkv, D, page, sb, qt):
    rng = np.random.default_rng(Hq + D + page)
    P = 5 * page if page < 128 else 2 * page
    for B in (1, 3, 21):
        lens = [P + int(x) for x in rng.integers(0, 3 * page, B)]
        lens[0] = P  # nothing of its own
        if B > 2:
            lens[1], lens[2] = P - page - 5, 0  # shorter than the prefix; empty
        N = P // page + sum(max(-(-n // page) - P // page, 0) for n in lens) + 1
        tables = random_tables(rng, lens, page, N, P // page + 4, P // page)
        pages = make_pool(rng, N, Hkv, page, D, sb)
        spoil(pages, tables, lens, page)
        tables[1:, :P // page] = 12345  # the other tables' entries there are not read
        q, qf = queries(rng, (B, Hq, D), qt)
        got = pg.sdpa_int4_paged(q, *map(dev, pages), dev(tables), ints(lens), Hq // Hkv, 0.9, shared_prefix=P)
        close(host(got), OP.sdpa_int4_paged(qf, pages, tables, lens, page, Hq // Hkv, 0.9, shared_prefix=P), f"B {B}")


@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 2, 128, 32), (4, 2, 256, 64), (8, 1, 512, 32)])
@pytest.mark.parametrize("window,sinks", [(50, 0), (200, 5), (30, 150), (300, 64), (700, 300)])
def test_shared_prefix_with_window_and_sinks(pg, Hq, Hkv, D, page, window, sinks):
    rng = np.random.default_rng(window)
    P, B = 8 * page, 9
    lens = [P + int(x) for x in rng.integers(0, 4 * page, B)]
    lens[3], lens[4] = P // 2 + 3, P
    wins = [window] * B
    wins[5] = 0
    N = P // page + sum(max(-(-n // page) - P // page, 0) for n in lens)
    tables = random_tables(rng, lens, page, N, P // page + 4, P // page)
    tables[0, 3] = -1  # and one page of the prefix missing
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    spoil(pages, tables, lens, page)
    q, qf = queries(rng, (B, Hq, D), "bf16")
    got = pg.sdpa_int4_paged(q, *map(dev, pages), dev(tables), ints(lens), Hq // Hkv, 1.0, 0, sinks, windows=ints(wins),
                             shared_prefix=P)
    close(host(got), OP.sdpa_int4_paged(qf, pages, tables, lens, page, Hq // Hkv, 1.0, 0, sinks, windows=wins,
                                        shared_prefix=P))


def test_shared_prefix_long(pg):
    rng = np.random.default_rng(77)
    Hq, Hkv, D, page, P, B = 4, 2, 256, 64, 4096, 12
    lens = [P + int(x) for x in rng.integers(1, 900, B)]
    N = P // page + sum(-(-n // page) - P // page for n in lens)
    tables = random_tables(rng, lens, page, N, -(-max(lens) // page), P // page)
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    q, qf = queries(rng, (B, Hq, D), "bf16")
    args = (q, *map(dev, pages), dev(tables), ints(lens), 2, 1.0)
    got = pg.sdpa_int4_paged(*args, shared_prefix=P)
    close(host(got), OP.sdpa_int4_paged(qf, pages, tables, lens, page, 2))
    apart = pg.sdpa_int4_paged(*args)
    close(host(apart), host(got))
    assert torch.equal(got, pg.sdpa_int4_paged(*args, shared_prefix=P))


@pytest.mark.parametrize("Hq,Hkv,D,page", [(2, 1, 128, 32), (16, 4, 128, 64), (4, 2, 256, 32), (8, 1, 256, 64),
                                           (6, 2, 256, 64), (2, 2, 512, 32), (8, 1, 512, 128)])
@pytest.mark.parametrize("prior,new,window,sinks", [(0, 1, 0, 0), (0, 70, 0, 0), (31, 2, 0, 0), (97, 66, 50, 0),
                                                    (200, 40, 33, 4), (130, 150, 64, 70), (500, 3, 100, 33)])
def test_prompt(pg, Hq, Hkv, D, page, prior, new, window, sinks):
    rng = np.random.default_rng(prior + new)
    n = prior + new
    N = -(-n // page) + 1
    table = random_tables(rng, [n], page, N, N + 1)
    sb, qt = [("f16", "bf16"), ("f32", "f32"), ("f16", "f32"), ("f32", "f16")][(Hq + prior) % 4]
    pages = make_pool(rng, N, Hkv, page, D, sb)
    spoil(pages, table, [n], page)
    q, qf = queries(rng, (new, Hq, D), qt)
    got = pg.sdpa_int4_paged_prefill(q, *map(dev, pages), dev(table[0]), prior, Hq // Hkv, 0.9, window, sinks)
    close(host(got), OP.sdpa_int4_paged_prefill(qf, pages, table[0], prior, page, Hq // Hkv, 0.9, window, sinks))


@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 2, 128, 32), (4, 2, 256, 64), (4, 2, 512, 32), (2, 1, 256, 32)])
def test_prompt_masked_values_and_bad_pages(pg, Hq, Hkv, D, page):
    """A row's result does not depend on NaN or infinite keys it does not attend,
    though others of its block do; missing pages take their keys along."""
    rng = np.random.default_rng(9)
    prior, new, W, sinks = 150, 90, 40, 5
    n = prior + new
    N = -(-n // page)
    table = random_tables(rng, [n], page, N, N)
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    for t, bad in ((n - 1, np.nan), (n - 2, np.inf), (prior - W, -np.inf), (60, np.nan)):
        for i in (1, 2, 4, 5):
            pages[i][table[0, t // page], :, t % page] = bad
    q, qf = queries(rng, (new, Hq, D), "bf16")
    got = host(pg.sdpa_int4_paged_prefill(q, *map(dev, pages), dev(table[0]), prior, Hq // Hkv, 1.0, W, sinks))
    with np.errstate(all="ignore"):
        ref = OP.sdpa_int4_paged_prefill(qf, pages, table[0], prior, page, Hq // Hkv, 1.0, W, sinks)
    close(got[:new - 2], ref[:new - 2])  # query 0 attends t > prior - W
    pages = make_pool(rng, N, Hkv, page, D, "f32")
    for i in (1, 2, 4, 5):
        pages[i][0] = np.nan
    table[0][table[0] == 0] = -1
    table[0, -1] = N
    got = host(pg.sdpa_int4_paged_prefill(q, *map(dev, pages), dev(table[0]), prior, Hq // Hkv, 1.0, W, sinks))
    close(got, OP.sdpa_int4_paged_prefill(qf, pages, table[0], prior, page, Hq // Hkv, 1.0, W, sinks))


@pytest.mark.parametrize("Hq,Hkv,D,page,prior,new,W,sinks", [
    (4, 2, 256, 64, 3000, 150, 0, 0), (4, 2, 256, 64, 3000, 150, 1000, 4), (8, 1, 512, 64, 2000, 40, 0, 0),
    (2, 1, 128, 32, 4000, 9, 0, 0)])
def test_prompt_long(pg, Hq, Hkv, D, page, prior, new, W, sinks):
    rng = np.random.default_rng(prior)
    n = prior + new
    N = -(-n // page)
    table = random_tables(rng, [n], page, N, N)
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    q, qf = queries(rng, (new, Hq, D), "bf16")
    args = (q, *map(dev, pages), dev(table[0]), prior, Hq // Hkv, 1.0, W, sinks)
    got = pg.sdpa_int4_paged_prefill(*args)
    close(host(got), OP.sdpa_int4_paged_prefill(qf, pages, table[0], prior, page, Hq // Hkv, 1.0, W, sinks))
    assert torch.equal(got, pg.sdpa_int4_paged_prefill(*args))


def of_heads(pages, heads, gqa):
    """The pages of the kv heads of some query heads, one each."""
    return [x[:, [h // gqa for h in heads]] for x in pages]


# More workgroups of 64 rows than compute units: workgroups of 128 rows are taken.
MANY = [(66, 33, 256, 32), (33, 33, 256, 64), (66, 33, 128, 32)]


@pytest.mark.parametrize("sb,qt", [("f16", "bf16"), ("f32", "f32"), ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("Hq,Hkv,D,page", MANY)
@pytest.mark.parametrize("prior,window,sinks", [(0, 0, 0), (37, 70, 6), (130, 31, 100)])
def test_prompt_of_many_heads(pg, Hq, Hkv, D, page, prior, window, sinks, sb, qt):
    rng = np.random.default_rng(prior + Hq + D)
    new = 301 if Hq > Hkv else 650
    n = prior + new
    N = -(-n // page)
    table = random_tables(rng, [n], page, N, N + 1)
    pages = make_pool(rng, N, Hkv, page, D, sb)
    if window:  # keys that some rows do not attend: of one key each NaN, infinite
        pages[4][table[0, 120 // page], :, 120 % page] = np.nan
        pages[5][table[0, (n - 1) // page], :, (n - 1) % page] = np.inf
        table[0, 5] = -1
    spoil(pages, table, [n], page)
    q, qf = queries(rng, (new, Hq, D), qt)
    got = host(pg.sdpa_int4_paged_prefill(q, *map(dev, pages), dev(table[0]), prior, Hq // Hkv, 0.9, window, sinks))
    heads = [0, 1, Hq // 2, Hq - 1]
    with np.errstate(all="ignore"):
        ref = OP.sdpa_int4_paged_prefill(qf[:, heads], of_heads(pages, heads, Hq // Hkv), table[0], prior, page, 1, 0.9,
                                         window, sinks)
    keep = np.isfinite(ref).all((1, 2))
    assert keep.sum() >= (new // 2 if window else new)
    close(got[:, heads][keep], ref[keep])


@pytest.mark.parametrize("sb,qt", [("f16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("D", [128, 256])
def test_shared_prefix_of_many_heads(pg, D, sb, qt):
    rng = np.random.default_rng(D)
    Hkv, Hq, page, B = 66, 132, 32, 130
    P = 5 * page
    lens = [P + int(x) for x in rng.integers(0, 2 * page, B)]
    lens[7], lens[99] = P - page - 5, 0
    N = P // page + sum(max(-(-n // page) - P // page, 0) for n in lens)
    tables = random_tables(rng, lens, page, N, P // page + 2, P // page)
    pages = make_pool(rng, N, Hkv, page, D, sb)
    spoil(pages, tables, lens, page)
    q, qf = queries(rng, (B, Hq, D), qt)
    got = pg.sdpa_int4_paged(q, *map(dev, pages), dev(tables), ints(lens), 2, 0.9, 100, 3, shared_prefix=P)
    heads = [0, 67, 131]
    ref = OP.sdpa_int4_paged(qf[:, heads], of_heads(pages, heads, 2), tables, lens, page, 1, 0.9, 100, 3, shared_prefix=P)
    close(host(got)[:, heads], ref)


@pytest.mark.parametrize("scale", [0.0, -0.7])
def test_scale_zero_and_negative(pg, scale):
    rng = np.random.default_rng(3)
    for Hq, Hkv, D, page in ((4, 2, 256, 64), (8, 1, 512, 32), (2, 1, 128, 32)):
        lens = [200, 77, 0]
        N = 15
        tables = random_tables(rng, lens, page, N, 7)
        pages = make_pool(rng, N, Hkv, page, D, "f16")
        q, qf = queries(rng, (3, Hq, D), "bf16")
        d = [dev(p) for p in pages]
        for P in (0, page):
            t = tables.copy()
            t[1:, :P // page] = t[0, :P // page]
            got = pg.sdpa_int4_paged(q, *d, dev(t), ints(lens), Hq // Hkv, scale, shared_prefix=P)
            close(host(got), OP.sdpa_int4_paged(qf, pages, t, lens, page, Hq // Hkv, scale))
        got = pg.sdpa_int4_paged_prefill(q, *d, dev(tables[0]), 190, Hq // Hkv, scale)
        close(host(got), OP.sdpa_int4_paged_prefill(qf, pages, tables[0], 190, page, Hq // Hkv, scale))


def test_offsets_past_32_bits(pg):
    """Pages behind the pool's first 4 GiB."""
    Hq, Hkv, D, page = 8, 4, 512, 1024
    N = 4200  # 1 MiB a page of K
    rng = np.random.default_rng(12)
    kq = torch.empty((N, Hkv, page, D // 8), dtype=torch.int32, device="cuda")
    sc = torch.empty((N, Hkv, page, D // 64), dtype=torch.float16, device="cuda")
    pool = [kq, sc, torch.empty_like(sc), torch.empty_like(kq), torch.empty_like(sc), torch.empty_like(sc)]
    at = [N - 1, N - 2]
    small = make_pool(rng, 2, Hkv, page, D, "f16")
    for t, s in zip(pool, small):
        for i, p in enumerate(at):
            x = dev(s[i])
            t[p] = x.view(torch.int32) if x.dtype == torch.uint32 else x
    pool = [t.view(torch.uint32) if t.dtype == torch.int32 else t for t in pool]
    q, qf = queries(rng, (1, Hq, D), "bf16")
    table, mine = ints([at]), np.array([[0, 1]])
    close(host(pg.sdpa_int4_paged(q, *pool, table, ints([1500]), 2)), OP.sdpa_int4_paged(qf, small, mine, [1500], page, 2))
    close(host(pg.sdpa_int4_paged(q, *pool, table, ints([1500]), 2, shared_prefix=1024)),
          OP.sdpa_int4_paged(qf, small, mine, [1500], page, 2))
    close(host(pg.sdpa_int4_paged_prefill(q, *pool, table[0], 1499, 2)),
          OP.sdpa_int4_paged_prefill(qf, small, mine[0], 1499, page, 2))
    new = rng.standard_normal((2, 1, Hkv, 40, D)).astype(np.float32)
    pg.kv_append_int4_paged(dev(new[0]), dev(new[1]), *pool, table, ints([1010]))
    OP.append(small, new[0], new[1], mine, [1010], page, "f16")
    for t, s in zip(pool, small):
        assert np.array_equal(host((t.view(torch.int32) if t.dtype == torch.uint32 else t)[at]).view(s.dtype), s)
    pg.kv_pages_copy(pool, ints([N - 1]), ints([0]))
    for t, s in zip(pool, small):
        assert np.array_equal(host(t[0]), s[0])


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("mode", ["mlx", "minmax"])
@pytest.mark.parametrize("B,Hkv,T,D,page,sb,xt", [(3, 2, 1, 128, 32, "f16", "bf16"), (4, 1, 70, 256, 32, "f32", "f32"),
                                                  (2, 3, 129, 512, 64, "f16", "f16"), (1, 2, 33, 64, 128, "f32", "f32")])
def test_append(pg, B, Hkv, T, D, page, sb, xt, mode):
    rng = np.random.default_rng(T)
    N, width = 20, 5
    tables = rng.permutation(N)[:B * width].reshape(B, width).astype(np.int32)
    tables[0, 1] = -1
    tables[-1, 2] = N
    pos = [int(x) for x in rng.integers(0, page * 2, B)]
    pos[-1] = width * page - 20  # runs past the table
    if B > 2:
        pos[1] = -3
    pages = make_pool(rng, N, Hkv, page, D, sb)
    k, kf = queries(rng, (B, Hkv, T, D), xt)
    v, vf = queries(rng, (B, Hkv, T, D), xt)
    d = [dev(p) for p in pages]
    pg.kv_append_int4_paged(k, v, *d, dev(tables), ints(pos), mode=mode)
    want = [p.copy() for p in pages]
    OP.append(want, kf, vf, tables, pos, page, sb, mode)
    for got, ref in zip(d, want):
        assert np.array_equal(host(got).view(np.uint8), ref.view(np.uint8))


# ---------------------------------------------------------------------------
# page operations
# ---------------------------------------------------------------------------

def random_state(rng, S, width, N, page, full=0.6):
    """Sequences with pages of their own and shared ones; pages in random order."""
    order = list(rng.permutation(N))
    tables = np.full((S, width), -1, np.int32)
    lens = np.zeros(S, np.int32)
    refs = np.zeros(N, np.int32)
    for s in range(S):
        if rng.random() > full:
            continue
        n = int(rng.integers(1, width * page + 1))
        k = -(-n // page)
        if k > len(order):
            continue
        tables[s, :k] = [order.pop() for _ in range(k)]
        lens[s] = n
    for e in tables[tables >= 0]:
        refs[e] += 1
    return tables, lens, refs


def pool_tensors(rng, L, N, Hkv, page, D):
    w = rng.integers(0, 2**32, (2, L, N, Hkv, page, D // 8), dtype=np.uint32)
    s = rng.standard_normal((4, L, N, Hkv, page, D // 64)).astype(np.float16)
    return [w[0], s[0], s[1], w[1], s[2], s[3]]


def same_state(pool, tables, refs, lens, pages, what):
    assert np.array_equal(host(tables), pool.tables), what
    assert np.array_equal(host(refs), pool.refs), what
    if lens is not None:
        assert np.array_equal(host(lens), pool.lengths), what
    for g, w in zip(pages, pool.pages):
        assert np.array_equal(host(g), w), what


@pytest.mark.parametrize("S,width,N,page", [(1, 1, 1, 32), (5, 4, 12, 32), (40, 9, 300, 32), (33, 70, 5000, 64),
                                            (1500, 3, 9000, 32)])
def test_reserve_fork_free_evict_compact(pg, S, width, N, page):
    """A random life of a pool, call by call against the oracle."""
    rng = np.random.default_rng(S)
    L, Hkv, D = (2, 1, 128) if N < 1000 else (1, 1, 64)
    page_data = pool_tensors(rng, L, N, Hkv, page, D) if N < 1000 else pool_tensors(rng, 1, N, 1, 32, 64)
    page = page if N < 1000 else 32
    tables, lens, refs = random_state(rng, S, width, N, page)
    pool = OP.Pool(tables, refs, lens, page, page_data)
    t, r, n, d = dev(tables), dev(refs), dev(lens), [dev(p) for p in page_data]
    for step in range(8):
        kind = ["reserve", "fork", "evict", "free", "fork", "compact", "reserve", "compact"][step]
        if kind == "reserve":
            ask = np.where(rng.random(S) < 0.5, rng.integers(-3, 3 * page, S), 0).astype(np.int32)
            got = pg.kv_pages_reserve(t, r, n, dev(ask), page)
            want = pool.reserve(ask)
            assert np.array_equal(host(got), want), (step, kind)
            grown = np.where(want == 1, np.maximum(ask, 0), 0).astype(np.int32)
            n += dev(grown)
            pool.lengths = (pool.lengths + grown).astype(np.int32)
        elif kind == "fork":
            par = np.where(rng.random(S) < 0.6, rng.integers(-1, S + 2, S), -1).astype(np.int32)
            got = pg.kv_pages_fork(d, t, r, n, dev(par))
            assert np.array_equal(host(got), pool.fork(par)), (step, kind)
        elif kind == "evict":
            which = (rng.random(S) < 0.7).astype(np.int32)
            pg.kv_pages_evict(t, r, n, page, page + 3, 5, dev(which))
            pool.evict(page + 3, 5, which)
        elif kind == "free":
            which = (rng.random(S) < 0.4).astype(np.int32)
            pg.kv_pages_free(t, r, n, dev(which))
            pool.free(which)
        else:
            before = (t.clone(), r.clone()) if step < 6 else (t, r)
            t2, r2, live = pg.kv_pages_compact(d, t, r, out=None if step < 6 else (t, r))
            assert int(live) == pool.compact()
            if step < 6:
                assert torch.equal(before[0], t) and torch.equal(before[1], r)  # inputs stay
            t, r = t2, r2
        same_state(pool, t, r, n, d, (step, kind))


def test_pages_run_out_in_order(pg):
    page, N = 32, 5
    tables, lens, refs = np.full((6, 4), -1, np.int32), np.zeros(6, np.int32), np.zeros(N, np.int32)
    refs[2] = 1
    pool = OP.Pool(tables, refs, lens, page)
    t, r, n = dev(tables), dev(refs), dev(lens)
    ask = np.array([33, 0, 65, 1, 129, 1], np.int32)  # two pages, none, three (refused), then none either
    assert host(pg.kv_pages_reserve(t, r, n, dev(ask), page)).tolist() == [1, 0, 0, 0, 0, 0]
    pool.reserve(ask)
    same_state(pool, t, r, n, [], "reserve")
    assert host(pg.kv_pages_reserve(t, r, n, ints([31, 64, 0, 0, 0, 0]), page)).tolist() == [1, 1, 0, 0, 0, 0]
    same_state(OP.Pool([[0, 1, -1, -1], [3, 4, -1, -1]] + [[-1] * 4] * 4, [1] * 5, lens, page), t, r, n, [], "last pages")


def test_copy_skips_what_is_no_page(pg):
    rng = np.random.default_rng(1)
    pages = pool_tensors(rng, 3, 10, 2, 64, 256)
    d = [dev(p) for p in pages]
    pg.kv_pages_copy(d, ints([1, 4, -1, 10, 7, 3]), ints([8, 4, 2, 5, 10, 0]))
    for g, w in zip(d, pages):
        w[:, 8], w[:, 0] = w[:, 1], w[:, 3]
        assert np.array_equal(host(g), w)


# ---------------------------------------------------------------------------
# together, streams, graphs
# ---------------------------------------------------------------------------

def reference_step(rng, cache_pages, pool, qf, knew, vnew, page, W, sinks, P=0):
    OP.append(cache_pages, knew, vnew, pool.tables, pool.lengths, page, "f16")
    return OP.sdpa_int4_paged(qf, cache_pages, pool.tables, pool.lengths + knew.shape[2], page, qf.shape[1] // knew.shape[1],
                              1.0, W, sinks, shared_prefix=P)


def test_a_serving_run(pg):
    """Two prompts, forks of them, decode steps with sinks and with the shared
    prefix, evictions, an ending, a packing -- every result against the oracle."""
    rng = np.random.default_rng(99)
    Hq, Hkv, D, page, S, N = 8, 4, 128, 32, 6, 60
    c = pg.PagedInt4KVCache(N, page, S, 12, Hkv, D, "cuda", num_layers=2)
    pool = OP.Pool(np.full((S, 12), -1, np.int32), np.zeros(N, np.int32), np.zeros(S, np.int32), page,
                   [host(t) for t in c.tensors()])
    layer = lambda i: [p[i] for p in pool.pages]  # noqa: E731

    def advance(n):
        c.advance(ints(n))
        pool.lengths = (pool.lengths + np.array(n)).astype(np.int32)

    for s, T in ((0, 100), (1, 64)):
        ask = np.zeros(S, np.int32)
        ask[s] = T
        assert host(c.reserve(ints(ask)))[s] == pool.reserve(ask)[s] == 1
        for i in range(2):
            k, kf = queries(rng, (Hkv, T, D), "bf16")
            v, vf = queries(rng, (Hkv, T, D), "bf16")
            c.append_one(i, s, k, v)
            OP.append(layer(i), kf[None], vf[None], pool.tables[s:s + 1], pool.lengths[s:s + 1], page, "f16")
            q, qf = queries(rng, (T, Hq, D), "bf16")
            got = c.prefill(i, s, q, 0, 2, 1.0, 40, 3)
            close(host(got), OP.sdpa_int4_paged_prefill(qf, layer(i), pool.tables[s], 0, page, 2, 1.0, 40, 3))
        advance(ask)
    par = np.array([-1, -1, 0, 0, 0, 1], np.int32)
    assert np.array_equal(host(c.fork(ints(par))), pool.fork(par))
    for step in range(40):
        ones = np.ones(S, np.int32)
        if step == 30:
            which = np.array([0, 1, 0, 0, 0, 1], np.int32)
            c.free(ints(which))
            pool.free(which)
            assert int(c.compact()) == pool.compact()
        if step >= 30:
            ones[[1, 5]] = 0
        assert np.array_equal(host(c.reserve(ints(ones))), pool.reserve(ones))
        for i in range(2):
            k, kf = queries(rng, (S, Hkv, 1, D), "bf16")
            v, vf = queries(rng, (S, Hkv, 1, D), "bf16")
            q, qf = queries(rng, (S, Hq, D), "bf16")
            W, sinks = ((0, 0), (50, 4))[i]
            c.append(i, k, v)
            got = c.attend(i, q, 2, 1.0, W, sinks)
            ref = reference_step(rng, layer(i), pool, qf, kf, vf, page, W, sinks)
            close(host(got), ref, f"step {step} layer {i}")
        advance(ones)
        same_state(pool, c.block_tables, c.refs, c.lengths, c.tensors(), step)
        if step == 20:
            # the four continuations of the first prompt share its three full pages
            some = [0, 2, 3, 4]
            q, qf = queries(rng, (4, Hq, D), "f16")
            got = pg.sdpa_int4_paged(q, *c.layer(0), c.block_tables[some], c.lengths[some], 2, shared_prefix=96)
            close(host(got), OP.sdpa_int4_paged(qf, layer(0), pool.tables[some], pool.lengths[some], page, 2))
    c.evict(50, 4)
    pool.evict(50, 4)
    same_state(pool, c.block_tables, c.refs, c.lengths, c.tensors(), "evict")


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 256), (8, 1, 512)])
def test_step_in_a_graph(pg, Hq, Hkv, D):
    """reserve + append + attend + advance, captured once and replayed: each
    replay is the next token; eager work lies between the replays."""
    page, S, N = 32, 3, 200
    rng = np.random.default_rng(D)

    def fresh():
        c = pg.PagedInt4KVCache(N, page, S, 30, Hkv, D, "cuda")
        first = ints([600, 333, 0])
        c.reserve(first)
        g = torch.Generator(device="cuda").manual_seed(4)
        k, v = (torch.randn((S, Hkv, 600, D), generator=g, device="cuda") for _ in range(2))
        c.append(0, k, v)
        c.advance(first)
        return c

    data = [[queries(rng, shape, "bf16")[0] for shape in ((S, Hkv, 1, D), (S, Hkv, 1, D), (S, Hq, D))] for _ in range(5)]
    ones = ints([1, 1, 1])

    def step(c, k, v, q):
        c.reserve(ones)
        c.append(0, k, v)
        out = c.attend(0, q, Hq // Hkv, 1.0, 300, 40, shared_prefix=0)
        c.advance(ones)
        return out

    eager = fresh()
    want = [step(eager, *x).clone() for x in data]
    c = fresh()
    bufs = [x.clone() for x in data[0]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    warm = fresh()
    with torch.cuda.stream(s):
        step(warm, *bufs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = step(c, *bufs)
    for x, w in zip(data, want):
        for b, y in zip(bufs, x):
            b.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
        step(warm, *data[1])  # eager work in between
    assert torch.equal(c.block_tables, eager.block_tables) and torch.equal(c.lengths, eager.lengths)


def test_two_graphs_with_workspaces_and_a_grown_one(pg):
    """Graphs captured with workspaces of their own run at once; a graph on the
    cached workspace stays right after a larger call has replaced it."""
    from gemma4metal_amd import _lib
    rng = np.random.default_rng(2)
    Hq, Hkv, D, page, B = 8, 4, 256, 64, 2
    lens = [5000, 4000]
    N = sum(-(-n // page) for n in lens)
    tables = random_tables(rng, lens, page, N, 80)
    pages = [dev(p) for p in make_pool(rng, N, Hkv, page, D, "f16")]
    t, n = dev(tables), ints(lens)
    qs = [queries(rng, (B, Hq, D), "bf16")[0] for _ in range(3)]
    want = [pg.sdpa_int4_paged(q, *pages, t, n, 2) for q in qs]
    size = _lib.load().tq_sdpa_int4_paged_workspace_size(B, Hq, Hkv, D, 80 * page, 0)
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs, outs = [], []
    ws = [torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda") for _ in range(2)] + [None]
    torch.cuda.synchronize()
    for q, s, w in zip(qs, streams, ws):
        pg.sdpa_int4_paged(q, *pages, t, n, 2, workspace=w, stream=s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(pg.sdpa_int4_paged(q, *pages, t, n, 2, workspace=w))
        graphs.append(g)
    big = queries(rng, (60, Hq, D), "bf16")[0]
    pg.sdpa_int4_paged(big, *pages, t[:1].expand(60, -1).contiguous(), n[:1].expand(60).contiguous(), 2,
                       stream=streams[2])
    junk = [torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda") for _ in range(30)]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
    assert all(int(j.min()) == int(j.max()) == 7 for j in junk)


def test_a_stream_of_ones_own(pg):
    rng = np.random.default_rng(6)
    Hq, Hkv, D, page = 4, 2, 128, 32
    tables = random_tables(rng, [700], page, 22, 22)
    pages = make_pool(rng, 22, Hkv, page, D, "f16")
    q, qf = queries(rng, (1, Hq, D), "bf16")
    d = [dev(p) for p in pages]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = pg.sdpa_int4_paged(q, *d, dev(tables), ints([700]), 2, stream=s)
    s.synchronize()
    close(host(got), OP.sdpa_int4_paged(qf, pages, tables, [700], page, 2))


def test_python_refusals(pg):
    rng = np.random.default_rng(0)
    d = [dev(p) for p in make_pool(rng, 4, 2, 32, 128, "f16")]
    q = torch.zeros((1, 4, 128), device="cuda")
    t, n = ints([[0, 1]]), ints([40])
    ok = lambda **k: pg.sdpa_int4_paged(k.get("q", q), *k.get("d", d), k.get("t", t), k.get("n", n), k.get("g", 2))  # noqa: E731
    ok()
    for bad in (dict(q=q[0]), dict(q=q.int()), dict(q=q.transpose(0, 1)), dict(t=t.long()), dict(t=t[0]), dict(n=n.float()),
                dict(n=ints([1, 2])), dict(d=[d[0], d[1].float()] + d[2:]), dict(d=d[:3] + [d[3][:2]] + d[4:]),
                dict(d=[d[0].float()] + d[1:]), dict(d=[x[:, :, ::2] for x in d]), dict(t=t.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            ok(**bad)
    from gemma4metal_amd._lib import TQError
    with pytest.raises(TQError, match="num_heads"):
        ok(g=4)
    with pytest.raises(TQError, match="shared_prefix"):
        pg.sdpa_int4_paged(q, *d, t, n, 2, shared_prefix=33)
    with pytest.raises(TQError, match="max_kv_len"):
        pg.sdpa_int4_paged(q, *d, t, n, 2, max_kv_len=65)
    with pytest.raises(ValueError, match="workspace"):
        pg.kv_pages_reserve(t, ints([0] * 4), n, n, 32, workspace=torch.zeros(4, dtype=torch.uint8, device="cuda"))
