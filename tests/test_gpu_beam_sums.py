"""GPU: the sums of exponentials behind the choice of beams, where many logits are equal and
all err alike, and where logits are large."""
import numpy as np
import pytest
import torch

from tests.gpu_util import host
from tests.test_gpu_beam import _DT, check

pytestmark = pytest.mark.gpu

# A sum's error: a power of two off by an ulp (2^-23 of it at most), four steps of a sum in
# 32 bits.  A total's is that and, where it is near 0, little else (squares of 2^-20, roundings
# of corrections of that size): 1% for it.
SUM = 1.01 * (2.0**-23 + 4 * 2.0**-24)


@pytest.fixture(scope="module")
def bm():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from gemma4metal_amd import beam
    return beam


def plateaus(dtype, tops, V, every):
    """Rows with one largest logit in `every` tokens and all others alike, 5 to 15 below; the
    scores that bring the best totals near 0; those totals, in 64 bits."""
    rows = []
    rng = np.random.default_rng(V)
    for top in tops:
        for d in np.arange(5, 15.5, 0.5 if V > 100000 else 0.125):
            x = np.full(V, top - d, np.float32)
            x[[at + rng.integers(min(every, V - at)) for at in range(0, V, every)]] = top
            rows.append(x)
    t = torch.from_numpy(np.stack(rows))[:, None].to(_DT[dtype]).cuda()
    x = t[:, 0].float().cpu().numpy().astype(np.float64)
    most = x.max(1)
    less = np.log(np.exp(x - most[:, None]).sum(1))
    scores = less.astype(np.float32)
    return t, scores, scores.astype(np.float64) - less


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,every", [(4096, 1024), (32769, 1024), (262144, 1024), (5000, 4096), (70001, 70001), (1000, 100)])
def test_equal_logits(bm, dtype, V, every):
    x, scores, want = plateaus(dtype, (0.0, 3.71875, 14.25, -40.5), V, every)
    got = host(bm.beam_select(x, torch.from_numpy(scores)[:, None].cuda(), 1)[0])[:, 0].astype(np.float64)
    assert np.abs(got - want).max() <= SUM


@pytest.mark.parametrize("dtype,V", [("bf16", 32768), ("f32", 5000), ("f16", 262144)])
def test_beams_that_differ_by_little(bm, dtype, V):
    """A beam of equal logits beside one with a single token: in the order of their totals,
    as near as twice what a sum can be off."""
    x, scores, want = plateaus(dtype, (0.0, 14.25), V, 1024)
    only = torch.full_like(x, -np.inf)
    only[:, :, 7] = 1.0
    near = 2 * SUM
    for sign in (-1, 1):
        beside = (want + sign * near).astype(np.float32)
        both = torch.from_numpy(np.stack([scores, beside], 1)).cuda()
        parents = host(bm.beam_select(torch.cat([x, only], 1), both, 1)[1])[:, 0]
        assert np.array_equal(parents, 2 * np.arange(len(scores)) + (sign > 0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_logits(bm, dtype):
    """Rows around 1,023, 1,025, far below 0, near the ends of fp32, and rows whose parts lie
    on both sides of that."""
    rng = np.random.default_rng(2)
    V = 9000
    x = 3 * rng.standard_normal((10, V))
    x[1] += 1023
    x[2] += 1040
    x[3] -= 1030
    x[4] *= 500
    x[5] *= 1e30
    x[6] = -3e38
    x[7, 4096:] += 2000
    x[8, :5000] -= 5000
    x[9, :4096] = -np.inf
    t = torch.from_numpy(x.astype(np.float32)).to(_DT[dtype]).cuda()[:, None]
    scores = np.zeros((10, 1), np.float32)
    check(bm.beam_select(t, torch.from_numpy(scores).cuda(), 5), t.float().cpu().numpy(), scores, 5)
