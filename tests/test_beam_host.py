"""Beam search and batched chunks without a GPU: the oracle against closed forms, what
the C calls refuse before any GPU work, workspace sizes, and the C++ API's exports and
refusals."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from gemma4metal_amd import _lib
from oracle import beam as OB
from oracle import paged as OP

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EXE = os.path.join(ROOT, "tests", "cpp", "test_beam")
NULL, FAKE = None, 0x10000  # aligned, never dereferenced: validation fails first
F16, F32, BF16 = _lib.TQ_F16, _lib.TQ_F32, _lib.TQ_BF16


def refused(name, args, status, needle):
    lib = _lib.load()
    st = getattr(lib, name)(*args)
    msg = lib.tq_last_error().decode()
    assert st == status and needle in msg, (st, msg)


def select(**o):
    a = dict(x=FAKE, dt=BF16, gs=400, bs=100, sc=FAKE, fin=NULL, G=2, W=4, V=100, K=4, pad=0, so=FAKE, po=FAKE, to=FAKE,
             ws=FAKE, wb=1 << 20) | o
    return "tq_beam_select", list(a.values()) + [NULL]


def pages(**o):
    six = (ctypes.c_void_p * 6)(*[FAKE] * 6)
    a = dict(six=six, sb=F16, L=1, Hkv=2, D=128, t=FAKE, r=FAKE, n=FAKE, p=FAKE, g=FAKE, S=4, P=3, N=12, page=32, ws=FAKE,
             wb=1 << 20) | o
    return "tq_kv_pages_reorder", list(a.values()) + [NULL]


def rows(**o):
    a = dict(kq=FAKE, ks=FAKE, kb=FAKE, vq=FAKE, vs=FAKE, vb=FAKE, sb=F16, B=4, Hkv=2, D=128, cap=40, n=FAKE, p=FAKE,
             ws=FAKE, wb=1 << 20) | o
    return "tq_kv_reorder_int4", list(a.values()) + [NULL]


def chunks(**o):
    a = dict(q=FAKE, dt=BF16, kq=FAKE, ks=FAKE, kb=FAKE, vq=FAKE, vs=FAKE, vb=FAKE, sb=F16, out=FAKE, B=2, N=6, Hq=4, Hkv=2,
             D=128, page=32, num=12, t=FAKE, P=100, st=FAKE, sl=FAKE, new=6, kv=3000, gqa=2, scale=1.0, W=0, sinks=0,
             ws=FAKE, wb=1 << 40) | o
    return "tq_sdpa_int4_paged_chunks", list(a.values()) + [NULL]


@pytest.mark.parametrize("call,status,needle", [
    (select(dt=7), 1, "x_dtype"), (select(G=-1), 1, "groups"), (select(W=0), 1, "beams"), (select(W=65), 1, "beams"),
    (select(K=0), 1, "num_out"), (select(K=65), 1, "num_out"), (select(V=0), 1, "vocab"), (select(V=(1 << 24) + 1), 1, "vocab"),
    (select(pad=100), 1, "pad_token"), (select(pad=-1), 1, "pad_token"), (select(x=NULL), 1, "null"), (select(sc=NULL), 1, "null"),
    (select(to=NULL), 1, "null"), (select(bs=-1), 1, "strides"), (select(x=FAKE + 1), 1, "aligned"),
    (select(ws=NULL), 4, "workspace"), (select(wb=8), 4, "workspace"), (select(ws=FAKE + 8), 1, "16-byte"),
    (select(G=1 << 20, W=64, V=1 << 20, wb=1 << 60), 1, "too large"),
    (pages(page=48), 2, "page_size"), (pages(S=65537), 1, "num_seqs"), (pages(sb=BF16), 1, "sb_dtype"), (pages(six=None), 1, "null"),
    (pages(p=NULL), 1, "null"), (pages(g=NULL), 1, "null"), (pages(wb=64), 4, "workspace"), (pages(ws=FAKE + 4), 1, "16-byte"),
    (pages(D=100), 1, "head_dim"), (pages(P=0), 1, "max_pages"),
    (rows(sb=BF16), 1, "sb_dtype"), (rows(B=1025), 1, "batch"), (rows(B=-1), 1, "batch"), (rows(D=100), 1, "head_dim"),
    (rows(cap=0), 1, "kv_capacity"), (rows(kq=NULL), 1, "null"), (rows(vb=FAKE + 2), 1, "aligned"), (rows(n=NULL), 1, "null"),
    (rows(wb=16), 4, "workspace"), (rows(ws=FAKE + 8), 1, "16-byte"), (rows(Hkv=0), 1, "num_kv_heads"),
    (rows(B=1024, Hkv=65535, cap=1 << 24), 1, "too large"),
    (chunks(B=65536), 1, "batch"), (chunks(N=-1), 1, "queries"), (chunks(new=-1), 1, "max_new"), (chunks(dt=9), 1, "q_dtype"),
    (chunks(D=64), 2, "head_dim"), (chunks(gqa=3), 1, "num_heads"), (chunks(W=-1), 1, "sliding_window"),
    (chunks(scale=float("inf")), 1, "scale"), (chunks(st=NULL), 1, "null"), (chunks(sl=NULL), 1, "null"),
    (chunks(kv=3201), 1, "max_kv_len"), (chunks(kv=-1), 1, "max_kv_len"), (chunks(q=FAKE + 8), 1, "aligned"),
    (chunks(out=NULL), 1, "null"), (chunks(ws=NULL), 4, "workspace"), (chunks(wb=1000), 4, "workspace"),
    (chunks(ws=FAKE + 8), 1, "16-byte"), (chunks(N=1 << 29), 1, "too many"),
])
def test_refused_before_any_gpu_work(call, status, needle):
    refused(*call, status, needle)


def test_nothing_to_do():
    lib = _lib.load()
    for name, args in (select(G=0, x=NULL, ws=NULL), pages(S=0, t=NULL, ws=NULL), rows(B=0, kq=NULL, ws=NULL),
                       chunks(B=0, q=NULL, ws=NULL), chunks(N=0, q=NULL, ws=NULL)):
        assert getattr(lib, name)(*args) == 0, (name, lib.tq_last_error())


def test_workspace_sizes():
    lib = _lib.load()
    f = lib.tq_beam_select_workspace_size
    assert f(0, 1, 1) == 0 and 0 < f(1, 1, 1) <= f(1, 1, 5000) < f(1, 2, 5000) < f(3, 2, 5000)
    assert lib.tq_kv_reorder_int4_workspace_size(1025) == 0 and lib.tq_kv_reorder_int4_workspace_size(4) > 0
    g = lib.tq_kv_pages_reorder_workspace_size
    assert g(4, 10, 3) > lib.tq_kv_pages_workspace_size(4, 10) and g(4, 10, 0) == 0
    h = lib.tq_sdpa_int4_paged_chunks_workspace_size
    assert h(4, 8, 4, 2, 128, 2, 100) == 0 and h(4, 8, 4, 2, 128, 2, 5000) > 0 and h(4, 8, 4, 3, 128, 2, 5000) == 0
    # it does not shrink with longer bounds
    for new in (1, 8, 40, 300):
        last = 0
        for kv in (64, 512, 600, 4096, 100000):
            assert h(3, 600, 32, 16, 256, new, kv) >= last
            last = h(3, 600, 32, 16, 256, new, kv)


def test_oracle_select_closed_forms():
    x = np.zeros((1, 2, 4), np.float32)
    x[0, 1, 2] = np.log(5.0)              # of 8 in all
    val, par, tok = OB.beam_select(x, np.zeros((1, 2), np.float32), 3)
    assert par.tolist() == [[1, 0, 0]] and tok.tolist() == [[2, 0, 1]]
    assert np.allclose(val, np.log([5 / 8, 1 / 4, 1 / 4]), atol=1e-7)
    x[0, 0, 3] = np.inf
    val, par, tok = OB.beam_select(x, np.array([[-1.0, -np.inf]], np.float32), 2, pad=1)
    assert par.tolist() == [[0, -1]] and tok.tolist() == [[3, -1]] and val[0, 0] == -1 and val[0, 1] == -np.inf
    val, par, tok = OB.beam_select(x, np.array([[-1.0, -3.0]], np.float32), 3, np.array([[0, 1]]), 1)
    assert tok.tolist() == [[3, 1, -1]] and par.tolist() == [[0, 1, -1]]


def test_oracle_reorder_keeps_counts_and_rows():
    rng = np.random.default_rng(3)
    S, page, N = 6, 32, 40
    tables, lens = np.full((S, 4), -1, np.int32), rng.integers(0, 100, S).astype(np.int32)
    order = iter(rng.permutation(N))
    refs = np.zeros(N, np.int32)
    for s in range(S):
        for e in range(-(-lens[s] // page)):
            tables[s, e] = next(order)
            refs[tables[s, e]] = 1
    pool = OP.Pool(tables, refs, lens, page, [rng.standard_normal((2, N, 1, page, 2))])

    def row(p, s):
        n = p.lengths[s]
        return [p.pages[0][:, p.tables[s, t // page], 0, t % page].tolist() for t in range(n)]
    for _ in range(20):
        parents = rng.integers(-1, S, S)
        old = [row(pool, s) for s in range(S)]
        granted = OB.reorder(pool, parents)
        for s in range(S):
            assert granted[s] == (parents[s] >= 0)
            assert row(pool, s) == (old[parents[s]] if parents[s] >= 0 else [])
        count = np.zeros(N, np.int32)
        for e in pool.tables.ravel():
            count[e] += e >= 0
        assert np.array_equal(count, pool.refs)


def test_cpp_exports_and_refusals():
    lib = os.path.join(ROOT, "gemma4metal_amd", "libturboquant_hip.so")
    out = subprocess.run(["nm", "-DC", "--defined-only", lib], capture_output=True, text=True, check=True).stdout
    for c in ("beam_select", "kv_reorder_int4", "kv_pages_reorder", "sdpa_int4_paged_chunks"):
        assert f"turboquant::{c}(" in out, c
    env = {**os.environ, "HIP_VISIBLE_DEVICES": "", "ROCR_VISIBLE_DEVICES": ""}
    r = subprocess.run([EXE, "refusals"], capture_output=True, text=True, timeout=60, env=env)
    assert r.returncode == 0 and r.stdout.count("PASS") == 14, r.stdout + r.stderr


@pytest.mark.gpu
def test_cpp_run():
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.count("PASS") == 4, r.stdout + r.stderr
