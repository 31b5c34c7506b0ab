"""CPU: calls of the paged cache beside those of ``test_paged_host.py``: refusals
before any GPU work, the arithmetic of the page plans, the Python layer."""
import ctypes

import numpy as np
import pytest

from gemma4metal_amd import _lib
from oracle import paged as OP

NULL = ctypes.c_void_p(0)
FAKE = ctypes.c_void_p(0x10000)  # aligned, never dereferenced: validation fails first


# ---------------------------------------------------------------------------
# advancing
# ---------------------------------------------------------------------------

def advance(**over):
    a = dict(tab=FAKE, lens=FAKE, new=FAKE, adv=FAKE, S=4, P=8, N=16, page=32)
    assert set(over) <= set(a)
    a.update(over)
    lib = _lib.load()
    return lib.tq_kv_pages_advance(*a.values(), NULL), lib.tq_last_error().decode()


@pytest.mark.parametrize("over,status,needle", [
    (dict(tab=NULL), 1, "null"), (dict(lens=NULL), 1, "null"), (dict(new=NULL), 1, "null"), (dict(adv=NULL), 1, "null"),
    (dict(page=48), 2, "page_size"), (dict(N=0), 1, "num_pages"), (dict(P=0), 1, "max_pages"), (dict(S=-1), 1, "num_seqs"),
])
def test_advance_refuses_bad_arguments_on_the_host(over, status, needle):
    st, msg = advance(**over)
    assert st == status and needle in msg, (st, msg)


def test_advance_of_no_sequences_is_no_error():
    assert advance(S=0, tab=NULL, lens=NULL)[0] == 0


def test_oracle_advances_only_rows_that_have_pages():
    p = OP.Pool([[0, 1, -1], [2, -1, -1], [-1] * 3, [3, 4, 5], [6, 99, -1]], np.ones(7, np.int32), [64, 20, 0, 90, 30], 32)
    assert list(p.advance([1, 12, 1, 6, 3])) == [0, 1, 0, 1, 0]  # 99: no page of the pool
    assert p.lengths.tolist() == [64, 32, 0, 96, 30]
    assert list(p.advance([0, 1, -5, 1, -7])) == [0, 0, 0, 0, 0]  # row 96 is past the table
    assert p.lengths.tolist() == [64, 32, 0, 96, 23]
