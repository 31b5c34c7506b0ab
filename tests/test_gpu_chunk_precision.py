"""GPU: attention of chunks of a batch to the precision that its arithmetic has, in every
form of its kernels."""
import numpy as np
import pytest
import torch

from oracle import paged as OP
from tests.gpu_util import dev, host
from tests.test_gpu_chunks import batch, run
from tests.test_gpu_paged import close, ints
from tests.test_gpu_paged_calls import TILES, definition, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pg():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from gemma4metal_amd import paged
    return paged


@pytest.mark.parametrize("qt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("sb", ["f16", "f32"])
@pytest.mark.parametrize("D", [128, 256, 512])
@pytest.mark.parametrize("Hq,Hkv,new,lens", [(4, 2, [3, 3], [500, 70]), (8, 1, [1, 1], [900, 31]), (4, 2, [1, 1], [33, 1]),
                                             (4, 2, [70, 1, 2], [300, 800, 65]), (8, 1, [90, 1], [2100, 64])])
def test_every_form(pg, Hq, Hkv, new, lens, D, sb, qt):
    """Few rows, many and both, each group of dims on its own."""
    rng = np.random.default_rng(D + len(new))
    q, qf, pages, tables, starts = batch(rng, new, lens, Hq, Hkv, D, 32, sb, qt)
    got = run(pg, q, pages, tables, starts, lens, Hq // Hkv, D**-0.5, max_new=max(new))
    for b, L in enumerate(lens):
        mine = slice(starts[b], starts[b + 1])
        ref = definition(qf[mine], pages, tables[b], range(L - new[b] + 1, L + 1), 32, Hq // Hkv, D**-0.5)
        for g in range(0, D, 64):
            within(got[mine], ref, TILES, f"sequence {b}, dims from {g}", slice(g, g + 64))


@pytest.mark.parametrize("sb,qt", [("f16", "bf16"), ("f16", "f32"), ("f32", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("D,rows", [(128, 128), (256, 32), (256, 48), (512, 16)])
def test_around_the_limits_of_few_rows(pg, D, rows, sb, qt):
    """Sequences of as many rows as the kernels part at, two more and two less, alone and
    side by side, with keys to be split and without."""
    rng = np.random.default_rng(D + rows)
    Hq, Hkv, page = 4, 2, 32
    at = rows // 2
    for new, lens in (([at - 1], [700]), ([at], [2600]), ([at + 1], [2600]), ([at - 1, at, at + 1, 1], [90, 1500, 2600, 400])):
        q, qf, pages, tables, starts = batch(rng, new, lens, Hq, Hkv, D, page, sb, qt)
        got = run(pg, q, pages, tables, starts, lens, 2, D**-0.5, max_new=max(new), max_kv_len=max(lens))
        for b, L in enumerate(lens):
            mine = slice(starts[b], starts[b + 1])
            ref = definition(qf[mine], pages, tables[b], range(L - new[b] + 1, L + 1), page, 2, D**-0.5)
            within(got[mine], ref, TILES, f"{new}: sequence {b}")


LOG2E = 1.4426950408889634

# (score in powers of two below the last keys', factor of the V scales and biases) of 128
# keys each, so that a wave that takes every fourth block of 32 meets all of them
FADES = {
    "f16": [[(-60, 1e4), (0, 1e-3)], [(-60, 1e4), (0, 1e-4)], [(-60, 1e4), (-40, 10.0), (-20, 1e-2), (0, 1e-4)],
            [(-60, 1e-4), (0, 1e4)]],
    "f32": [[(-60, 1e10), (0, 0.1)], [(-120, 1e25), (-80, 1e10), (0, 1e-5)], [(-110, 1e-20), (-90, 1e10), (0, 1e-10)],
            [(-60, 1e3), (-30, 1.0), (0, 1e-3)], [(-126, 1e20), (0, 1e-30)],
            [(-160, 1e20), (0, 1e-20)]],
}


@pytest.mark.parametrize("sb,qt,fade", [(sb, qt, i) for sb, qt in (("f16", "bf16"), ("f16", "f32"), ("f32", "f32"), ("f32", "f16"))
                                        for i in range(len(FADES[sb]))])
@pytest.mark.parametrize("D,new", [(128, 3), (128, 60), (128, 100), (256, 3), (256, 40), (512, 3), (512, 30)])
def test_keys_that_fade_leave_no_rounding(pg, D, new, sb, qt, fade):
    """What a row adds up is rounded against what is left of its sums, not against what
    they held before a larger score came.  What the first keys leave is at most 1e-4 of the
    result, so that their scores' rounding is no part of the error -- but in the case of 126,
    whose result they are as far as fp32 holds their weights (2^-126 and more: rows that are
    120 below at most): 2^-24 of 126 in each of four roundings (the sum, the factor, the
    product with it less the reference, fp32 queries), ln 2 of that in every weight."""
    rng = np.random.default_rng(D + new + fade)
    Hq, Hkv, page, lens = 4, 2, 32, [500]
    q, qf, pages, tables, starts = batch(rng, [new], lens, Hq, Hkv, D, page, sb, qt)
    q, qf = q.abs(), np.abs(qf)
    steps, scale = FADES[sb][fade], 1 / 128
    sums = qf.sum(-1)
    for t in range(lens[0]):
        e, r = tables[0, t // page], t % page
        far, factor = steps[min(t // 128, len(steps) - 1)]
        # (q . k) scale = far ln 2, but for the last keys' own spread
        if far:
            pages[1][e, :, r] = 0
            pages[2][e, :, r] = far / LOG2E / (scale * sums.mean())
        for i in (4, 5):
            pages[i][e, :, r] *= pages[i].dtype.type(factor)
    assert all(np.isfinite(p[tables[0, 0]].astype(np.float64)).all() for p in pages[1:3] + pages[4:])
    got = run(pg, q, pages, tables, starts, lens, Hq // Hkv, scale)
    ref = definition(qf, pages, tables[0], range(lens[0] - new + 1, lens[0] + 1), page, Hq // Hkv, scale)
    tol, rows = TILES, np.ones(sums.shape, bool)
    if steps[0][0] == -126:
        tol, rows = TILES + 4 * 126 * 2.0**-24 / LOG2E, 126 * sums / sums.mean() <= 120
    assert np.isfinite(got).all()
    if rows.any():
        within(got[rows], [ref[0][rows], ref[1][rows]], tol, f"{steps}")


@pytest.mark.parametrize("D,B", [(128, 1024), (128, 1025), (512, 2100), (256, 3000)])
def test_batches_of_several_launches(pg, D, B):
    """More sequences than a launch takes: chunks of either kind in all of them, a last
    launch whose keys are split, empty sequences, rows behind the last chunk; in a graph."""
    rng = np.random.default_rng(B)
    Hq, Hkv, page = 2, 1, 32
    new = rng.integers(0, 3, B)
    new[[3, B // 2, B - 1]] = [70, 140, 5]
    prior = rng.integers(0, 60, B)
    prior[[3, B - 1]] = [2500, 2600]
    lens = (new + prior).tolist()
    q, qf, pages, tables, starts = batch(rng, new.tolist(), lens, Hq, Hkv, D, page)
    extra = torch.cat([q, q[:3]])
    args = [extra, *[dev(p) for p in pages], dev(tables), ints(starts), ints(lens), 2, D**-0.5]
    out = torch.full(extra.shape, 7.0, device="cuda")
    kw = dict(max_new=140, max_kv_len=max(lens), out=out)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        pg.sdpa_int4_paged_chunks(*args, **kw)
    s.synchronize()
    first = host(out)
    ref = OP.sdpa_int4_paged_chunks(qf, pages, tables, starts, lens, page, 2, D**-0.5)
    close(first[:starts[-1]], ref)
    assert (first[starts[-1]:] == 7).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        pg.sdpa_int4_paged_chunks(*args, **kw)
    for _ in range(3):
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(host(out), first)
