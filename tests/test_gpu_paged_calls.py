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


def test_sequences_that_append_nothing(pg):
    """With a count per sequence the others attend just their own rows, whatever
    lies behind those."""
    rng = np.random.default_rng(12)
    Hq, Hkv, D, page = 4, 2, 128, 32
    c = pg.PagedInt4KVCache(6, page, 3, 2, Hkv, D, "cuda")
    first = ints([40, 33, 7])
    c.reserve(first)
    for s, T in enumerate((40, 33, 7)):
        k, v = (queries(rng, (Hkv, 64, D), "bf16")[0] for _ in range(2))
        c.append_one(0, s, k, v)  # rows behind the length too
    c.advance(first)
    q, qf = queries(rng, (3, Hq, D), "bf16")
    n = ints([0, 1, 0])
    got = host(c.attend(0, q, 2, new=n))
    ref = OP.sdpa_int4_paged(qf, [host(x[0]) for x in c.tensors()], host(c.block_tables), [40, 34, 7], page, 2)
    close(got, ref)


# ---------------------------------------------------------------------------
# prefixes whose sequences give pages up
# ---------------------------------------------------------------------------

def shared_run(pg, rng, Hq, Hkv, D, page, P, tails):
    """A prompt of P rows, forked, each sequence with rows of its own; the cache and
    its state on the host."""
    S, width = len(tails), P // page + 4
    N = P // page + 4 * S
    c = pg.PagedInt4KVCache(N, page, S, width, Hkv, D, "cuda")
    ask = np.zeros(S, np.int32)
    ask[0] = P
    assert host(c.reserve(ints(ask)))[0] == 1
    c.append_one(0, 0, *(queries(rng, (Hkv, P, D), "bf16")[0] for _ in range(2)))
    c.advance(ints(ask))
    par = np.zeros(S, np.int32)
    par[0] = -1
    assert host(c.fork(ints(par))).tolist() == [0] + [1] * (S - 1)
    assert host(c.reserve(ints(tails))).all()
    for s, T in enumerate(tails):
        c.append_one(0, s, *(queries(rng, (Hkv, T, D), "bf16")[0] for _ in range(2)))
    assert host(c.advance(ints(tails))).all()
    return c


def attention_of(c, qf, gqa, W, sinks):
    return OP.sdpa_int4_paged(qf, [host(x[0]) for x in c.tensors()], host(c.block_tables), host(c.lengths), c.page_size,
                              gqa, 1.0, W, sinks)


CASES = [(4, 2, 128, 32, 5), (8, 1, 256, 64, 4), (8, 1, 512, 32, 9), (4, 2, 512, 128, 2)]


@pytest.mark.parametrize("Hq,Hkv,D,page,blocks", CASES)
def test_a_prefix_outlives_the_sequence_it_came_with(pg, Hq, Hkv, D, page, blocks):
    rng = np.random.default_rng(D + page)
    P, none = blocks * page, ints([0] * 4)
    c = shared_run(pg, rng, Hq, Hkv, D, page, P, [9, 40, 1, 2 * page])
    q, qf = queries(rng, (4, Hq, D), "bf16")
    whole = attention_of(c, qf, Hq // Hkv, 0, 0)
    close(host(c.attend(0, q, Hq // Hkv, new=none, shared_prefix=P)), whole)
    c.free(ints([1, 0, 0, 0]))
    for table in (c.block_tables[2, :blocks], c.prefix_table(P), c.prefix_table(P, torch.tensor([1, 3], device="cuda"))):
        got = host(c.attend(0, q, Hq // Hkv, new=none, shared_prefix=P, prefix_table=table))
        close(got[1:], whole[1:])
        assert not got[0].any()


@pytest.mark.parametrize("Hq,Hkv,D,page,blocks", CASES)
@pytest.mark.parametrize("sinks", [0, 5])
def test_a_prefix_after_evictions(pg, Hq, Hkv, D, page, blocks, sinks):
    """The longest sequence comes first and gives up what the others attend."""
    rng = np.random.default_rng(D + sinks)
    P, W, none = blocks * page, blocks * page - page // 2, ints([0] * 4)
    c = shared_run(pg, rng, Hq, Hkv, D, page, P, [3 * page, 40, 1, page])
    q, qf = queries(rng, (4, Hq, D), "bf16")
    whole = attention_of(c, qf, Hq // Hkv, W, sinks)
    c.evict(W, sinks)
    tables = host(c.block_tables)[:, :blocks]
    assert (tables[0] < 0).sum() > (tables[2] < 0).sum()
    close(attention_of(c, qf, Hq // Hkv, W, sinks), whole)  # nothing attended was given up
    got = c.attend(0, q, Hq // Hkv, 1.0, W, sinks, new=none, shared_prefix=P, prefix_table=c.prefix_table(P))
    close(host(got), whole)


def test_prefix_table_refusals(pg):
    rng = np.random.default_rng(0)
    d = [dev(p) for p in make_pool(rng, 4, 2, 32, 128, "f16")]
    q = torch.zeros((1, 4, 128), device="cuda")
    t, n = ints([[0, 1]]), ints([40])
    pg.sdpa_int4_paged(q, *d, t, n, 2, shared_prefix=32, prefix_table=t[0, :1])
    for bad in (t[0], t[0, :0], t[0, :1].long(), t[0, :1].cpu(), t[:, :1]):
        with pytest.raises(ValueError, match="prefix_table"):
            pg.sdpa_int4_paged(q, *d, t, n, 2, shared_prefix=32, prefix_table=bad)


# ---------------------------------------------------------------------------
# page plans
# ---------------------------------------------------------------------------

def test_reserve_of_more_pages_than_32_bits_count(pg):
    """1,024 neighbours that need 2^31 pages together (tables of 8 GiB, all empty): the
    first request is small and granted, the others are refused, and nothing else
    changes."""
    S, width, page, N = 1024, (1 << 21) + 2, 32, 9
    t = torch.full((S, width), -1, dtype=torch.int32, device="cuda")
    r, n = ints([1, 0, 1] + [0] * 6), ints([0] * S)
    ask = torch.full((S,), width * page, dtype=torch.int32, device="cuda")
    ask[0], ask[1] = 33, 0
    got = host(pg.kv_pages_reserve(t, r, n, ask, page))
    assert got[0] == 1 and not got[1:].any()
    assert host(r).tolist() == [1, 1, 1, 1] + [0] * 5 and host(t[0, :3]).tolist() == [1, 3, -1]
    assert int(t[0, 2:].max()) == -1 and int(t[1:].amax(1).max()) == -1


def test_named_arguments_and_a_stream(pg):
    rng = np.random.default_rng(3)
    Hq, Hkv, D, page = 4, 2, 128, 32
    names = ("k_quant", "k_scales", "k_biases", "v_quant", "v_scales", "v_biases")
    d = dict(zip(names, map(dev, make_pool(rng, 4, Hkv, page, D, "f16"))))
    q = queries(rng, (1, Hq, D), "bf16")[0]
    t, n = ints([[2, 0, 3]]), ints([80])
    want = pg.sdpa_int4_paged(q, *d.values(), t, n, 2)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (None, s):
        got = pg.sdpa_int4_paged(queries=q, **d, block_tables=t, seq_lens=n, gqa_factor=2, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    pg.kv_pages_free(block_tables=t, refs=ints([1] * 4), lengths=n, which=ints([1]), stream=s)
    s.synchronize()
    assert host(t).tolist() == [[-1] * 3] and host(n).tolist() == [0]


# ---------------------------------------------------------------------------
# precision
# ---------------------------------------------------------------------------

# Errors are taken relative to mag = sum_t w_t |v_t|, the attention of the values'
# magnitudes (0.8 of sigma): a rounding of a weight or of a partial sum is relative to
# that, while the result itself may be as small as the values cancel.  2-norms over many
# outputs add roundings as independent ones, each uniform within half a step (rms 0.58
# of half a step).
#
# Weights.  Parts leave a remainder r, uniform within half a step, and the last part
# rounds that: an error of half of r's own step, which halves with every halving of r.
# - Decode, fp16 scales: two bf16 parts (8 bits), |r| <= 2^-8, |error| <= 2^-17, rms
#   sqrt(1/3 1/2 / (1 - 1/8)) = 0.44 of that in the weight's octave, 0.31 of the weight:
#   2.4e-6 of nibbles' distances from 7.5 (sigma), 3e-6 of mag for one key; but a
#   weight of 1 is exact, and two of a half are off by 2.1e-6.  Many average out.
# - Decode, fp32 scales: a third part, 2^-25.
# - Tiles: two fp16 parts (11 bits, the first truncated), |r| <= 2^-10, |error| <=
#   2^-22: 1.3e-7.  A group whose V scales are 2^-9 of the largest has weights of 2^-5
#   there and a last step of 2^-24: 0.58 2^-20 = 5.5e-7, 0.7e-6 of mag for one key.
# Decode's sums of (16 + n) s: 24 sigma / 3 = 8, 2^-24 8 0.58 = 0.3e-6 a step, 0.5e-6 over
# the few that count.
# Scores.  With scale 1 / sqrt D, |score| < 8 (log2 domain): 2^-24 8 0.58 of a rounding, 8
# of them: 0.8e-6, ln 2 of that in a weight.  With scale 1, < 86: 2.2e-6 each, 4 of them at
# that size, ln 2: 3e-6, of which p (1 - p) sqrt 2 <= 0.35 remain: 1e-6.
# Decode's queries: exact of 16 bits but for a few far below the largest.  fp32 in steps
# of 4.5 / 8.36e6: 0.29 sqrt D of that, 2.5e-6 (D 256), 3.5e-6 (D 512), 0.35 of it with
# scale 1, 1 / sqrt D of it else; heads as columns (D 512, GQA 8) 4.5 / 2.24e6: 13e-6,
# 4.6e-6 with scale 1, 0.6e-6 else.
# In all: scale 1 / sqrt D: fp16 scales 2.3e-6, fp32 0.95e-6, tiles 0.9e-6; scale 1: 2.6e-6
# (fp16), 1.7e-6 (fp32), heads as columns with fp32 queries 5.2e-6.  About 1.6 times that is
# allowed.  A part that got lost would be 2^-9 of a weight or more.
DECODE, DECODE_F32, TILES = 2.0**-18, 2.0**-19, 1.5e-6
DECODE_ONE, DECODE_ONE_COLUMNS = 2.0**-18, 2.0**-17


def definition(q, pages, table, n_of, page, gqa, scale, window=0, sinks=0):
    """Rows q [R, Hq, D] at positions n_of[r] - 1 of one sequence, in 64 bits: results,
    and the same of the values' magnitudes."""
    k, v, has = OP.rows(pages, table, page, max(n_of))
    out = np.zeros((2,) + q.shape)
    for h in range(q.shape[1]):
        s = float(np.float32(scale)) * (q[:, h].astype(np.float64) @ k[h // gqa].T)
        for r, n in enumerate(n_of):
            s[r, ~(OP.visible(n, max(n_of), window, sinks) & has)] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[0, :, h], out[1, :, h] = p @ v[h // gqa], p @ np.abs(v[h // gqa])
    return out


def within(got, ref_mag, tol, what, dims=None):
    d = slice(None) if dims is None else dims
    ref, mag = ref_mag[0][..., d], ref_mag[1][..., d]
    err = np.linalg.norm(got[..., d] - ref) / np.linalg.norm(mag)
    assert np.isfinite(err) and err <= tol, f"{what}: {err:.3e} of the magnitudes, {tol:.1e} allowed"


PRECISION = [(8, 4, 128, 32), (8, 1, 128, 64), (8, 4, 256, 64), (8, 1, 256, 32), (4, 2, 512, 64), (8, 1, 512, 128)]


@pytest.mark.parametrize("sb,qt", [("f16", "bf16"), ("f32", "f32"), ("f16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("Hq,Hkv,D,page", PRECISION)
def test_precision(pg, Hq, Hkv, D, page, sb, qt):
    """Decode, a shared prefix and a prompt, each to the error that its arithmetic has."""
    rng = np.random.default_rng(Hq + D)
    gqa, scale, P = Hq // Hkv, D**-0.5, 4 * 128
    lens = [P + 1, P + 61, P + 128, 1777]
    N = P // page + sum(-(-n // page) - P // page for n in lens)
    tables = random_tables(rng, lens, page, N, -(-max(lens) // page), P // page)
    pages = make_pool(rng, N, Hkv, page, D, sb)
    d = [dev(p) for p in pages]
    q, qf = queries(rng, (len(lens), Hq, D), qt)
    columns = D == 512 and gqa % 8 == 0 and qt == "f32"
    for sc, tol in ((scale, DECODE if sb == "f16" else DECODE_F32), (1.0, DECODE_ONE_COLUMNS if columns else DECODE_ONE)):
        refs = [definition(qf[b:b + 1], pages, tables[b], [n], page, gqa, sc) for b, n in enumerate(lens)]
        for shared in (0, P):
            got = host(pg.sdpa_int4_paged(q, *d, dev(tables), ints(lens), gqa, sc, shared_prefix=shared))
            for b, n in enumerate(lens):
                within(got[b:b + 1], refs[b], tol, f"decode of {n}, shared {shared}, scale {sc}")
    new, prior = 70, 1777 - 70
    q, qf = queries(rng, (new, Hq, D), qt)
    got = host(pg.sdpa_int4_paged_prefill(q, *d, dev(tables[3]), prior, gqa, scale))
    within(got, definition(qf, pages, tables[3], range(prior + 1, 1778), page, gqa, scale), TILES, "prompt")


def uneven_pool(rng, kind, N, Hkv, page, D, sb, table):
    """A pool whose V scales are not of one size: of groups, of the first rows, of rows
    in turn (N(0, 1) rows, their scales and biases times powers of two)."""
    k = O.quantize_int4(O.rms_norm(rng.standard_normal((N, Hkv, page, D)).astype(np.float32)), sb)
    x = rng.standard_normal((N, Hkv, page, D)).astype(np.float32)
    first = [(table[t // page], t % page) for t in range(96)]
    if kind == "first":  # zeros: the quantizer's least scale
        for e, r in first:
            x[e, :, r] = 0.0
    w, *sbs = O.quantize_int4(x, "f32")
    for y in sbs:
        if kind.startswith("group"):
            y[..., -1] *= np.float32(2.0**int(kind[5:]))
        elif kind.startswith("all"):
            y *= np.float32(2.0**int(kind[3:]))
        elif kind == "spread":
            y[..., 0] *= np.float32(2.0**30)
            y[..., 1] *= np.float32(2.0**-30)
        elif kind.startswith("rows"):
            even, odd = map(int, kind[4:].split("/"))
            y[:, :, ::2] *= np.float32(2.0**even)
            y[:, :, 1::2] *= np.float32(2.0**odd)
        elif kind == "zero":
            for e, r in first:
                y[e, :, r] = 0.0
    return list(k) + [w] + [y.astype({"f16": np.float16, "f32": np.float32}[sb]) for y in sbs]


UNEVEN = [("f16", "bf16", k) for k in ("group-8", "group-12", "group-16", "first", "zero", "rows-10/5", "all-14", "all10")] + \
         [("f32", "f32", k) for k in ("group-8", "group-12", "group-40", "first", "zero", "spread", "rows-30/30", "all-30", "all30")]


@pytest.mark.parametrize("sb,qt,kind", UNEVEN)
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 4, 128, 32), (4, 2, 256, 64), (8, 1, 512, 32)])
def test_unlike_v_scales(pg, Hq, Hkv, D, page, sb, qt, kind):
    """Each group of 64 values to its own magnitude, also where the scales of a tile or
    of tiles are far apart."""
    rng = np.random.default_rng(D + len(kind))
    gqa, scale, P = Hq // Hkv, D**-0.5, 256
    lens = [P + 190, P + 5, P + 77]
    N = P // page + sum(-(-n // page) - P // page for n in lens)
    tables = random_tables(rng, lens, page, N, -(-max(lens) // page), P // page)
    pages = uneven_pool(rng, kind, N, Hkv, page, D, sb, tables[0])
    d = [dev(p) for p in pages]
    groups = [slice(g, g + 64) for g in range(0, D, 64)]
    new, prior = 150, lens[0] - 150
    q, qf = queries(rng, (new, Hq, D), qt)
    got = host(pg.sdpa_int4_paged_prefill(q, *d, dev(tables[0]), prior, gqa, scale, 200, 70))
    ref = definition(qf, pages, tables[0], range(prior + 1, lens[0] + 1), page, gqa, scale, 200, 70)
    for g in groups:
        within(got, ref, TILES, f"prompt, dims {g.start}", g)
    q, qf = queries(rng, (len(lens), Hq, D), qt)
    for shared in (0, P):
        got = host(pg.sdpa_int4_paged(q, *d, dev(tables), ints(lens), gqa, scale, shared_prefix=shared))
        for b, n in enumerate(lens):
            ref = definition(qf[b:b + 1], pages, tables[b], [n], page, gqa, scale)
            for g in groups:
                within(got[b:b + 1], ref, DECODE if sb == "f16" else DECODE_F32,
                       f"decode of {n}, shared {shared}, dims {g.start}", g)


@pytest.mark.parametrize("sb,qt,kind", UNEVEN)
@pytest.mark.parametrize("Hq,Hkv,D,page", [(66, 33, 128, 32), (66, 33, 256, 32)])
def test_unlike_v_scales_128_rows(pg, Hq, Hkv, D, page, sb, qt, kind):
    rng = np.random.default_rng(D + len(kind))
    gqa, scale, new, prior = Hq // Hkv, D**-0.5, 301, 200  # (more workgroups of 64 rows than compute units)
    n = new + prior
    N = -(-n // page)
    table = random_tables(rng, [n], page, N, N)[0]
    pages = uneven_pool(rng, kind, N, Hkv, page, D, sb, table)
    q, qf = queries(rng, (new, Hq, D), qt)
    got = host(pg.sdpa_int4_paged_prefill(q, *map(dev, pages), dev(table), prior, gqa, scale))
    heads = [0, 1, Hq // 2, Hq - 1]
    some = [x[:, [h // gqa for h in heads]] for x in pages]
    ref = definition(qf[:, heads], some, table, range(prior + 1, n + 1), page, 1, scale)
    for g in range(0, D, 64):
        within(got[:, heads], ref, TILES, f"dims {g}", slice(g, g + 64))


# ---------------------------------------------------------------------------
# long sequences: their pages come from a small pool, many times each
# ---------------------------------------------------------------------------

def keys_of(n, window, sinks):
    """The keys that the query at n - 1 attends."""
    if window <= 0 or n <= window:
        return np.arange(n)
    return np.concatenate([np.arange(min(sinks, n - window)), np.arange(n - window, n)])


def counted(qf, pages, table, n, page, gqa, scale, window=0, sinks=0, heads=None):
    """One query [Hq, D] in 64 bits by how often each row of the pool occurs."""
    N = pages[0].shape[0]
    t = keys_of(n, window, sinks)
    e = table[t // page].astype(np.int64)
    has = (e >= 0) & (e < N)
    count = np.bincount((e * page + t % page)[has], minlength=N * page).astype(np.float64)
    out = []
    for h in range(qf.shape[0]) if heads is None else heads:
        k, v = (O.dequantize(*(x[:, h // gqa].reshape(N * page, -1) for x in pages[i:i + 3])) for i in (0, 3))
        s = float(np.float32(scale)) * (k @ qf[h].astype(np.float64))
        p = count * np.exp(s - s[count > 0].max())
        out.append((p / p.sum()) @ v)
    return np.array(out)


def alias_tables(rng, B, width, N):
    t = rng.integers(0, N, (B, width)).astype(np.int32)
    t[:, 1::97] = -1  # some missing
    return t


# (more than 64 blocks a wave: page numbers are loaded again in the loop.  Four waves a
# workgroup, eight, D 512 without and with heads as columns; chunks of the host and the
# device)
@pytest.mark.parametrize("B,Hq,Hkv,D,n,sb", [
    (1, 2, 1, 128, 3_100_013, "f16"), (1, 2, 1, 256, 3_100_013, "f32"), (1, 8, 1, 512, 3_100_013, "f16"),
    (1, 2, 2, 512, 2_100_031, "f16"), (70, 8, 4, 256, 90_001, "f16"), (70, 16, 4, 128, 90_017, "f32"),
    (70, 8, 1, 512, 90_000, "f32"), (70, 2, 1, 512, 60_033, "f32"), (64, 32, 16, 128, 45_000, "f16"),
    (48, 32, 16, 256, 45_011, "f32"), (64, 64, 8, 512, 45_000, "f16"), (64, 16, 8, 512, 45_007, "f16")])
def test_decode_of_many_blocks_a_wave(pg, B, Hq, Hkv, D, n, sb):
    rng = np.random.default_rng(n)
    page, N, gqa = 32, 500, Hq // Hkv
    tables = alias_tables(rng, B, -(-n // page) + 1, N)
    pages = make_pool(rng, N, Hkv, page, D, sb)
    lens = [n] + [int(x) for x in rng.integers(n // 2, n, B - 1)]
    q, qf = queries(rng, (B, Hq, D), "bf16")
    d, t = [dev(p) for p in pages], dev(tables)
    some = sorted({0, 1, B // 2, B - 1} & set(range(B)))
    for W, sinks in ((0, 0), (n // 2 + 5, 77)):
        got = host(pg.sdpa_int4_paged(q, *d, t, ints(lens), gqa, 0.7, W, sinks))
        for b in some:
            heads = sorted({0, Hq // 2, Hq - 1})
            close(got[b, heads], counted(qf[b], pages, tables[b], lens[b], page, gqa, 0.7, W, sinks, heads), f"{b} W {W}")


@pytest.mark.parametrize("Hq,Hkv,D,prior,new", [(66, 33, 256, 9000, 301), (66, 33, 128, 9000, 301), (64, 8, 512, 5000, 600),
                                                (160, 160, 256, 6007, 65), (33, 33, 256, 2000, 650)])
def test_prompts_of_many_tiles_a_workgroup(pg, Hq, Hkv, D, prior, new):
    rng = np.random.default_rng(D + new)
    page, N, gqa = 32, 60, Hq // Hkv
    table = alias_tables(rng, 1, -(-(prior + new) // page), N)[0]
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    q, qf = queries(rng, (new, Hq, D), "bf16")
    d = [dev(p) for p in pages]
    for W, sinks in ((0, 0), (4500, 130)):
        got = host(pg.sdpa_int4_paged_prefill(q, *d, dev(table), prior, gqa, 0.7, W, sinks))
        for i in (0, 31, new - 1):
            heads = [0, Hq // 2, Hq - 1]
            close(got[i, heads], counted(qf[i], pages, table, prior + i + 1, page, gqa, 0.7, W, sinks, heads), f"row {i}")


@pytest.mark.parametrize("Hq,Hkv,D", [(66, 33, 256), (8, 1, 512), (8, 4, 128)])
def test_prefixes_of_many_tiles_a_workgroup(pg, Hq, Hkv, D):
    rng = np.random.default_rng(D)
    page, N, gqa, B, P = 64, 60, Hq // Hkv, 150, 12800
    tables = alias_tables(rng, B, P // page + 3, N)
    tables[1:, :P // page] = tables[0, :P // page]
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    lens = [P + int(x) for x in rng.integers(0, 3 * page, B)]
    lens[4] = 77
    q, qf = queries(rng, (B, Hq, D), "bf16")
    got = host(pg.sdpa_int4_paged(q, *map(dev, pages), dev(tables), ints(lens), gqa, 0.7, shared_prefix=P))
    for b in (0, 4, 149):
        heads = [0, Hq // 2, Hq - 1]
        close(got[b, heads], counted(qf[b], pages, tables[b], lens[b], page, gqa, 0.7, heads=heads), f"sequence {b}")


@pytest.mark.parametrize("Hq,Hkv,D", [(2, 1, 128), (4, 2, 256), (8, 1, 512)])
def test_positions_near_the_last(pg, Hq, Hkv, D):
    """Tables that reach 2^31 - 2^16 rows: every call at their end."""
    rng = np.random.default_rng(D)
    page, N, gqa = 32, 40, Hq // Hkv
    last = 2**31 - 2**16
    tables = np.full((2, last // page), -1, np.int32)
    tables[:, :8], tables[:, -64:] = rng.integers(0, 20, (2, 8)), rng.integers(0, 20, (2, 64))
    tables[:, -2:] = [[20, 21], [22, 23]]
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    d, t = [dev(p) for p in pages], dev(tables)
    k, kf = queries(rng, (2, Hkv, 50, D), "bf16")
    v, vf = queries(rng, (2, Hkv, 50, D), "bf16")
    pos = [last - 40, last - 17]  # 10 and 33 rows fall behind the tables
    pg.kv_append_int4_paged(k, v, *d, t, ints(pos))
    for b in range(2):
        m = last - pos[b]
        OP.append(pages, kf[b:b + 1, :, :m], vf[b:b + 1, :, :m], tables[b:b + 1, -4:], [pos[b] - (last - 4 * page)], page, "f16")
    for x, y in zip(d, pages):
        assert np.array_equal(host(x).view(np.uint8), y.view(np.uint8))
    q, qf = queries(rng, (2, Hq, D), "bf16")
    lens, W, sinks = [last, last - 9], 1500, 200
    want = np.array([counted(qf[b], pages, tables[b], lens[b], page, gqa, 0.7, W, sinks) for b in range(2)])
    close(host(pg.sdpa_int4_paged(q, *d, t, ints(lens), gqa, 0.7, W, sinks)), want)
    close(host(pg.sdpa_int4_paged(q, *d, t, ints(lens), gqa, 0.7, 0, sinks, windows=ints([W, W]))), want)
    for b in range(2):
        one = pg.sdpa_int4_paged(q[b:b + 1], *d, t[b:b + 1], ints(lens[b:b + 1]), gqa, 0.7, W, sinks)
        close(host(one)[0], want[b])
    many, mf = queries(rng, (70, Hq, D), "bf16")
    got = host(pg.sdpa_int4_paged_prefill(many, *d, t[0], last - 70, gqa, 0.7, W, sinks))
    for i in (0, 69):
        close(got[i], counted(mf[i], pages, tables[0], last - 69 + i, page, gqa, 0.7, W, sinks))
    # bookkeeping
    n, r = ints([last - 40, last - 40]), ints(np.bincount(tables[tables >= 0], minlength=N))
    t[1, -1] = -1
    assert host(pg.kv_pages_reserve(t, r, n, ints([41, 40]), page)).tolist() == [0, 1]
    assert host(pg.kv_pages_advance(t, r, n, ints([41, 40]), page)).tolist() == [0, 1]
    assert host(n).tolist() == [last - 40, last]
    before = host(t)
    pg.kv_pages_evict(t, r, n, page, 100, 33)
    e = np.arange(last // page, dtype=np.int64)
    for b, length in enumerate((last - 40, last)):
        gone = (e * page >= 33) & ((e + 1) * page <= length - 100)
        assert np.array_equal(host(t[b]), np.where(gone, -1, before[b]))


@pytest.mark.parametrize("Hq,Hkv,D,page", [(16, 1, 512, 64), (24, 1, 512, 32), (12, 1, 512, 32), (5, 1, 512, 64), (16, 1, 256, 64),
                                           (7, 1, 256, 512), (32, 1, 128, 256), (12, 4, 128, 1024), (20, 2, 128, 128)])
@pytest.mark.parametrize("sb", ["f16", "f32"])
def test_other_head_ratios_and_page_sizes(pg, Hq, Hkv, D, page, sb):
    rng = np.random.default_rng(Hq + page)
    gqa, P = Hq // Hkv, 2 * page
    lens = [P + 70, P, 33, 0, P + 3 * page - 1]
    N = P // page + sum(max(-(-n // page) - P // page, 0) for n in lens)
    tables = random_tables(rng, lens, page, N, P // page + 3, P // page)
    pages = make_pool(rng, N, Hkv, page, D, sb)
    spoil(pages, tables, lens, page)
    d = [dev(p) for p in pages]
    q, qf = queries(rng, (len(lens), Hq, D), "f16")
    for W, sinks in ((0, 0), (100, 40)):
        ref = OP.sdpa_int4_paged(qf, pages, tables, lens, page, gqa, 0.7, W, sinks)
        for shared in (0, P):
            close(host(pg.sdpa_int4_paged(q, *d, dev(tables), ints(lens), gqa, 0.7, W, sinks, shared_prefix=shared)), ref)
        q2, qf2 = queries(rng, (37, Hq, D), "f32")
        got = host(pg.sdpa_int4_paged_prefill(q2, *d, dev(tables[4]), lens[4] - 37, gqa, 0.7, W, sinks))
        close(got, OP.sdpa_int4_paged_prefill(qf2, pages, tables[4], lens[4] - 37, page, gqa, 0.7, W, sinks))


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 256), (8, 1, 512)])
def test_shared_prefix_in_a_graph(pg, Hq, Hkv, D):
    """Tiles and the joining decode, captured with a workspace of their own and replayed
    between eager calls; the prefix's table, lengths and queries change in place."""
    from gemma4metal_amd import _lib
    rng = np.random.default_rng(D)
    page, P, B, gqa = 64, 1024, 5, Hq // Hkv
    lens = [P + int(x) for x in rng.integers(1, 200, B)]
    N = 40 + 2 * P // page
    tables = random_tables(rng, lens, page, N, P // page + 4, P // page)
    other = rng.permutation(N)[:P // page].astype(np.int32)
    pages = make_pool(rng, N, Hkv, page, D, "f16")
    d, t, n, prefix = [dev(p) for p in pages], dev(tables), ints(lens), dev(tables[0, :P // page])
    size = _lib.load().tq_sdpa_int4_paged_workspace_size(B, Hq, Hkv, D, tables.shape[1] * page, P)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    q = queries(rng, (B, Hq, D), "bf16")[0]
    call = lambda w: pg.sdpa_int4_paged(q, *d, t, n, gqa, shared_prefix=P, prefix_table=prefix, workspace=w)  # noqa: E731
    call(ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(ws)
    for step in range(4):
        q.copy_(queries(rng, (B, Hq, D), "bf16")[0])
        n.copy_(ints([P + int(x) for x in rng.integers(1, 200, B)]))
        prefix.copy_(dev(other if step % 2 else tables[0, :P // page]))
        want = call(None).clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("Hq,Hkv,D", [(2, 1, 128), (4, 2, 256), (4, 2, 512), (8, 1, 512)])
@pytest.mark.parametrize("e", [-110, 100])
@pytest.mark.parametrize("qt", ["bf16", "f32"])
def test_queries_far_from_one(pg, Hq, Hkv, D, e, qt):
    """Queries times 2^e under a scale of 2^-e / sqrt D are the queries themselves; one
    row is 0, and attends all keys alike."""
    rng = np.random.default_rng(D)
    page, gqa, n = 32, Hq // Hkv, 200
    table = random_tables(rng, [n], page, 9, 9)[0]
    pages = make_pool(rng, 9, Hkv, page, D, "f32")
    d, t = [dev(p) for p in pages], dev(table)
    q, qf = queries(rng, (30, Hq, D), qt)
    q[0, 0], qf[0, 0] = 0, 0
    q = (q.float() * 2.0**e).to(q.dtype)  # exact: a power of two
    scale = float(np.float32(D**-0.5)) * 2.0**-e
    ref = definition(qf, pages, table, [n - 29 + i for i in range(30)], page, gqa, D**-0.5)
    within(host(pg.sdpa_int4_paged_prefill(q, *d, t, n - 30, gqa, scale)), ref, TILES, "prompt")
    lens = ints([n - 29 + i for i in range(30)])
    for shared in (0, 96):
        got = host(pg.sdpa_int4_paged(q, *d, t[None].expand(30, -1).contiguous(), lens, gqa, scale, shared_prefix=shared))
        within(got, ref, DECODE_F32, f"decode, shared {shared}")
