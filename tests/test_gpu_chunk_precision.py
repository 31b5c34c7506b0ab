"""GPU: attention of chunks of a batch to the precision that its arithmetic has, in every
form of its kernels."""
import numpy as np
import pytest
import torch

from tests.test_gpu_chunks import batch, run
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
