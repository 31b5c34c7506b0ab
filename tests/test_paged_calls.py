"""CPU: calls of the paged cache beside those of ``test_paged_host.py``: refusals
before any GPU work, the arithmetic of the page plans, the Python layer."""
import ctypes
import inspect
import os
import subprocess

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


# ---------------------------------------------------------------------------
# a prefix by a table of its own
# ---------------------------------------------------------------------------

def prefix(**over):
    a = dict(q=FAKE, qd=_lib.TQ_BF16, kq=FAKE, ks=FAKE, kb=FAKE, vq=FAKE, vs=FAKE, vb=FAKE, sb=_lib.TQ_F16, out=FAKE,
             B=2, Hq=32, Hkv=16, D=256, page=64, N=10, tab=FAKE, P=4, lens=FAKE, win=NULL, mx=256, gqa=2, scale=1.0,
             W=0, sinks=0, table=FAKE, pre=64, ws=NULL, wsb=0)
    assert set(over) <= set(a)
    a.update(over)
    lib = _lib.load()
    return lib.tq_sdpa_int4_paged_prefix(*a.values(), NULL), lib.tq_last_error().decode()


@pytest.mark.parametrize("over,status,needle", [
    (dict(pre=32), 1, "shared_prefix"), (dict(pre=320), 1, "shared_prefix"), (dict(pre=-64), 1, "shared_prefix"),
    (dict(lens=NULL), 1, "seq_lens"), (dict(tab=NULL), 1, "null"), (dict(D=64), 2, "head_dim"), (dict(mx=257), 1, "max_kv_len"),
    (dict(), 4, "workspace"),
])
def test_prefix_call_refuses_bad_arguments_on_the_host(over, status, needle):
    st, msg = prefix(**over)
    assert st == status and needle in msg and "tq_sdpa_int4_paged_prefix" in msg, (st, msg)


def test_prefix_call_with_nothing_to_do_is_no_error():
    assert prefix(B=0, q=NULL, table=NULL)[0] == 0


# ---------------------------------------------------------------------------
# page plans
# ---------------------------------------------------------------------------

def test_plans_of_more_pages_than_32_bits_count():
    r = subprocess.run([os.path.join(os.path.dirname(__file__), "cpp", "test_page_plan")], capture_output=True, text=True,
                       timeout=60)
    assert r.returncode == 0 and r.stdout.count("PASS") == 6, r.stdout + r.stderr


# ---------------------------------------------------------------------------
# the Python layer
# ---------------------------------------------------------------------------

FUNCTIONS = ["kv_append_int4_paged", "sdpa_int4_paged", "sdpa_int4_paged_prefill", "kv_pages_reserve",
             "kv_pages_advance", "kv_pages_fork", "kv_pages_free", "kv_pages_evict", "kv_pages_compact", "kv_pages_copy"]


@pytest.mark.parametrize("name", FUNCTIONS)
def test_every_argument_can_be_named(name):
    """Also the first: the call reaches the function's own checks (of host tensors)."""
    import torch
    from gemma4metal_amd import paged
    fn = getattr(paged, name)
    params = inspect.signature(fn).parameters
    assert params["stream"].kind is inspect.Parameter.KEYWORD_ONLY
    t = torch.zeros(1, dtype=torch.int32)
    args = {n: 32 if n in ("page_size", "sliding_window", "gqa_factor", "n_prior") else [t] * 6 if n == "pages" else t
            for n, p in params.items() if p.default is inspect.Parameter.empty}
    assert list(args) == list(params)[:len(args)]
    for call in (lambda: fn(**args), lambda: fn(*args.values()),
                 lambda: fn(*list(args.values())[:1], **dict(list(args.items())[1:]))):
        with pytest.raises(ValueError, match="must be on a GPU device"):
            call()
    with pytest.raises(TypeError, match=list(args)[0]):
        fn()
