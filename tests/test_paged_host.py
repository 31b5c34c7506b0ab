"""CPU: the paged cache's refusals (before any GPU call), its workspace sizes,
and the oracle that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

from gemma4metal_amd import _lib
from oracle import oracle as O
from oracle import paged as OP

NULL = ctypes.c_void_p(0)
FAKE = ctypes.c_void_p(0x10000)  # aligned, never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x10008)


def attend(**over):
    a = dict(q=FAKE, qd=_lib.TQ_BF16, kq=FAKE, ks=FAKE, kb=FAKE, vq=FAKE, vs=FAKE, vb=FAKE, sb=_lib.TQ_F16, out=FAKE,
             B=2, Hq=32, Hkv=16, D=256, page=64, N=10, tab=FAKE, P=4, lens=FAKE, win=NULL, mx=256, gqa=2, scale=1.0,
             W=0, sinks=0, pre=0, ws=NULL, wsb=0)
    assert set(over) <= set(a)
    a.update(over)
    lib = _lib.load()
    return lib.tq_sdpa_int4_paged(*list(a.values())[:-2], a["ws"], a["wsb"], NULL), lib.tq_last_error().decode()


def prompt(**over):
    a = dict(q=FAKE, qd=_lib.TQ_BF16, kq=FAKE, ks=FAKE, kb=FAKE, vq=FAKE, vs=FAKE, vb=FAKE, sb=_lib.TQ_F16, out=FAKE,
             Hq=32, Hkv=16, D=256, page=64, N=10, tab=FAKE, P=4, prior=100, new=70, gqa=2, scale=1.0, W=0, sinks=0,
             ws=NULL, wsb=0)
    assert set(over) <= set(a)
    a.update(over)
    lib = _lib.load()
    return lib.tq_sdpa_int4_paged_prefill(*list(a.values())[:-2], a["ws"], a["wsb"], NULL), lib.tq_last_error().decode()


COMMON = [
    (dict(D=100), 2, "head_dim"), (dict(D=64), 2, "head_dim"), (dict(Hq=30), 1, "num_heads"),
    (dict(qd=7), 1, "q_dtype"), (dict(sb=_lib.TQ_BF16), 1, "sb_dtype"), (dict(W=-1), 1, "sliding_window"),
    (dict(sinks=-1), 1, "num_sinks"), (dict(scale=float("nan")), 1, "scale"), (dict(scale=float("inf")), 1, "scale"),
    (dict(page=16), 2, "page_size"), (dict(page=48), 2, "page_size"), (dict(page=2048), 2, "page_size"),
    (dict(N=0), 1, "num_pages"), (dict(P=0), 1, "max_pages"), (dict(P=1 << 26, page=64), 1, "2^31"),
    (dict(q=NULL), 1, "null"), (dict(tab=NULL), 1, "null"), (dict(out=NULL), 1, "null"), (dict(vb=NULL), 1, "null"),
    (dict(q=ODD), 1, "queries must be 16-byte"), (dict(ks=ODD), 1, "k_scales must be 16-byte"),
    (dict(out=ODD), 1, "out must be 16-byte"), (dict(gqa=0, Hq=0), 1, "gqa"),
]


@pytest.mark.parametrize("over,status,needle", COMMON + [
    (dict(lens=NULL), 1, "seq_lens"), (dict(mx=257), 1, "max_kv_len"), (dict(mx=-1), 1, "max_kv_len"),
    (dict(pre=32), 1, "shared_prefix"), (dict(pre=320), 1, "shared_prefix"), (dict(pre=-64), 1, "shared_prefix"),
    (dict(B=-1), 1, "batch"), (dict(B=70000), 1, "batch"),
])
def test_attention_refuses_bad_arguments_on_the_host(over, status, needle):
    st, msg = attend(**over)
    assert st == status and needle in msg, (st, msg)


@pytest.mark.parametrize("over,status,needle", COMMON + [
    (dict(prior=-1), 1, "n_prior"), (dict(new=-1), 1, "n_prior"), (dict(prior=200), 1, "exceeds"),
    (dict(new=70000, P=4096), 1, "65535"),
])
def test_prompt_attention_refuses_bad_arguments_on_the_host(over, status, needle):
    st, msg = prompt(**over)
    assert st == status and needle in msg, (st, msg)


@pytest.mark.parametrize("call", ["attend", "prompt"])
def test_refuses_tables_that_reach_past_whole_splits_in_32_bits(call):
    """Positions are rounded up in 32 bits: 2^31 - 2^16 rows are the most."""
    st, msg = {"attend": attend, "prompt": prompt}[call](P=(1 << 31) // 1024 - 63, page=1024)
    assert st == 1 and "2^31" in msg


def test_refuses_prompt_rows_past_32_bits():
    st, msg = prompt(Hq=65535, Hkv=1, gqa=65535, new=65535, prior=0, P=4096, page=64)
    assert st == 1 and "grid" in msg, msg


def test_nothing_to_do_is_no_error():
    assert attend(B=0, q=NULL, lens=NULL)[0] == 0
    assert prompt(new=0, q=NULL)[0] == 0


def plan(B, Hq, Hkv, D, n, W=0, sinks=0, P=0):
    lib = _lib.load()
    out = [ctypes.c_int(-1) for _ in range(4)]
    name = ctypes.create_string_buffer(64)
    assert lib.tq_sdpa_int4_paged_plan(B, Hq, Hkv, D, n, W, sinks, P, *map(ctypes.byref, out), name, 64) == 0
    return [x.value for x in out] + [name.value.decode()]


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 4, 128), (2, 1, 128), (32, 16, 256), (8, 1, 256), (32, 4, 512), (4, 2, 512)])
def test_every_plan_has_room(Hq, Hkv, D):
    """A split for every key that a sequence may attend, and a workspace that
    holds the splits of any window."""
    lib = _lib.load()
    for B in (1, 2, 7, 16, 64, 65, 300):
        for n in (0, 1, 33, 127, 128, 129, 192, 500, 1000, 4097, 20000, 131072, 1 << 20):
            for P in (0, 64, 4096):
                if P > n:
                    continue
                room = lib.tq_sdpa_int4_paged_workspace_size(B, Hq, Hkv, D, n, P)
                for W, sinks in ((0, 0), (1, 0), (64, 33), (100, 64), (1000, 4), (4000, 3000)):
                    splits, chunk, pre, device, _ = plan(B, Hq, Hkv, D, n, W, sinks, P)
                    most = n if W == 0 else min(n, W + 62 + -(-sinks // 32) * 32)
                    keys = -(-min(most, n - P) // 32) * 32
                    assert splits >= 1 and chunk >= 1 and chunk % 32 == 0
                    assert splits * chunk >= keys, (B, n, W, sinks, P)
                    assert (pre > 0) == (P > 0)
                    need = (1 << 18) + B * Hq * (splits + pre) * (D + 2) * 4
                    assert room >= need, (B, n, W, sinks, P, room, need)


def append(**over):
    a = dict(k=FAKE, v=FAKE, xd=_lib.TQ_F32, kq=FAKE, ks=FAKE, kb=FAKE, vq=FAKE, vs=FAKE, vb=FAKE, sb=_lib.TQ_F16, B=2,
             Hkv=16, D=256, page=64, N=10, tab=FAKE, P=4, pos=FAKE, T=1, mode=0)
    assert set(over) <= set(a)
    a.update(over)
    lib = _lib.load()
    return lib.tq_kv_append_int4_paged(*a.values(), NULL), lib.tq_last_error().decode()


@pytest.mark.parametrize("over,status,needle", [
    (dict(xd=5), 1, "x_dtype"), (dict(sb=_lib.TQ_BF16), 1, "sb_dtype"), (dict(mode=3), 1, "mode"),
    (dict(D=100), 1, "head_dim"), (dict(page=24), 2, "page_size"), (dict(N=0), 1, "num_pages"), (dict(B=-1), 1, "sizes"),
    (dict(tab=NULL), 1, "null"), (dict(pos=NULL), 1, "null"), (dict(k=ODD), 1, "k_new"), (dict(vs=ODD), 1, "page tensors"),
])
def test_append_refuses_bad_arguments_on_the_host(over, status, needle):
    st, msg = append(**over)
    assert st == status and needle in msg, (st, msg)


def test_page_calls_refuse_bad_arguments_on_the_host():
    lib = _lib.load()
    err = lambda: lib.tq_last_error().decode()  # noqa: E731
    six = (ctypes.c_void_p * 6)(*[0x10000] * 6)
    bad = (ctypes.c_void_p * 6)(*[0x10000] * 5 + [0x10008])
    hole = (ctypes.c_void_p * 6)(*[0x10000] * 5 + [0])
    big = 1 << 30
    assert lib.tq_kv_pages_reserve(FAKE, FAKE, FAKE, FAKE, FAKE, 4, 8, 16, 20, FAKE, big, NULL) == 2
    assert lib.tq_kv_pages_reserve(FAKE, FAKE, NULL, FAKE, FAKE, 4, 8, 16, 32, FAKE, big, NULL) == 1 and "null" in err()
    assert lib.tq_kv_pages_reserve(FAKE, FAKE, FAKE, FAKE, FAKE, 4, 8, 16, 32, FAKE, 8, NULL) == 4 and "workspace" in err()
    assert lib.tq_kv_pages_reserve(FAKE, FAKE, FAKE, FAKE, FAKE, 4, 8, 16, 32, ODD, big, NULL) == 1 and "aligned" in err()
    assert lib.tq_kv_pages_reserve(FAKE, FAKE, FAKE, FAKE, FAKE, -1, 8, 16, 32, FAKE, big, NULL) == 1
    fork = lambda pages, sb=_lib.TQ_F16, L=1, S=4: lib.tq_kv_pages_fork(  # noqa: E731
        pages, sb, L, 16, 256, FAKE, FAKE, FAKE, FAKE, FAKE, S, 8, 16, 32, NULL, 0, NULL)
    assert fork(bad) == 1 and "16-byte" in err()
    assert fork(hole) == 1 and "null" in err()
    assert fork(NULL) == 1 and "null" in err()
    assert fork(six, sb=_lib.TQ_BF16) == 1 and "sb_dtype" in err()
    assert fork(six, L=0) == 1 and "num_layers" in err()
    assert fork(six) == 4 and "workspace" in err()
    assert fork(six, S=0) == 0
    assert lib.tq_kv_pages_free(FAKE, FAKE, FAKE, NULL, 4, 8, 16, NULL) == 1 and "null" in err()
    assert lib.tq_kv_pages_free(FAKE, FAKE, FAKE, FAKE, 0, 8, 16, NULL) == 0
    assert lib.tq_kv_pages_evict(FAKE, FAKE, FAKE, NULL, 4, 8, 16, 32, 0, 4, NULL) == 1 and "sliding_window" in err()
    assert lib.tq_kv_pages_evict(FAKE, FAKE, FAKE, NULL, 4, 8, 16, 32, 8, -4, NULL) == 1 and "num_sinks" in err()
    assert lib.tq_kv_pages_compact(six, 1, 1, 16, 256, FAKE, FAKE, FAKE, FAKE, NULL, 4, 8, 16, 32, FAKE, big, NULL) == 1
    assert lib.tq_kv_pages_copy(six, 1, 1, 16, 256, 16, 32, FAKE, NULL, 3, NULL) == 1 and "null" in err()
    assert lib.tq_kv_pages_copy(six, 1, 1, 16, 256, 16, 32, FAKE, FAKE, -3, NULL) == 1
    assert lib.tq_kv_pages_copy(six, 1, 1, 16, 256, 16, 32, NULL, NULL, 0, NULL) == 0


def test_python_layer_refuses_host_tensors():
    import torch
    from gemma4metal_amd import paged
    t = torch.zeros((2, 2, 32, 16), dtype=torch.int32)
    s = torch.zeros((2, 2, 32, 2))
    with pytest.raises(ValueError, match="GPU"):
        paged.sdpa_int4_paged(torch.zeros((1, 2, 128)), t, s, s, t, s, s, torch.zeros((1, 2), dtype=torch.int32),
                              torch.zeros(1, dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="six"):
        paged.kv_pages_copy((t, s), torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


# ---------------------------------------------------------------------------
# the oracle
# ---------------------------------------------------------------------------

def small_pool(rng, N, Hkv, page, D, sb="f32"):
    k = O.quantize_int4(O.rms_norm(rng.standard_normal((N, Hkv, page, D)).astype(np.float32)), sb)
    v = O.quantize_int4(rng.standard_normal((N, Hkv, page, D)).astype(np.float32), sb)
    return list(k) + list(v)


@pytest.mark.parametrize("window", [0, 1, 40, 500])
def test_oracle_without_sinks_is_the_contiguous_rule(window):
    rng = np.random.default_rng(5)
    pages = small_pool(rng, 5, 2, 32, 128)
    table = np.array([[3, 0, 4, -1]], np.int32)
    q = rng.standard_normal((1, 4, 128)).astype(np.float32)
    flat = [np.concatenate([x[p] for p in (3, 0, 4)], 1) for x in pages]
    for n in (0, 1, 32, 33, 95):
        got = OP.sdpa_int4_paged(q, pages, table, [n], 32, 2, 0.3, window)
        ref = O.sdpa_int4(q[0], *[x[:, :n] for x in flat], 2, 0.3, window) if n else np.zeros((4, 128))
        np.testing.assert_allclose(got[0], ref, atol=1e-12)


def test_oracle_sinks_and_missing_pages():
    rng = np.random.default_rng(6)
    pages = small_pool(rng, 4, 1, 32, 128)
    q = rng.standard_normal((1, 1, 128)).astype(np.float32)
    full = OP.sdpa_int4_paged(q, pages, np.array([[0, 1, 2]]), [80], 32, 1)
    # sinks and window that cover everything are no restriction; one key is its row
    for W, s in ((80, 0), (30, 50), (50, 30), (1, 79)):
        np.testing.assert_allclose(OP.sdpa_int4_paged(q, pages, np.array([[0, 1, 2]]), [80], 32, 1, window=W, sinks=s),
                                   full, atol=1e-12)
    two = OP.sdpa_int4_paged(q, pages, np.array([[0, 9, 2]]), [80], 32, 1, window=1, sinks=1)
    k, v, _ = OP.rows(pages, [0, 1, 2], 32, 80)
    s = k[0][[0, 79]] @ q[0, 0].astype(np.float64)
    p = np.exp(s - s.max())
    np.testing.assert_allclose(two[0, 0], (p / p.sum()) @ v[0][[0, 79]], atol=1e-12)
    # no page, no key
    assert not OP.sdpa_int4_paged(q, pages, np.array([[-1, 4, 99]]), [80], 32, 1).any()
    assert not OP.sdpa_int4_paged(q, pages, np.array([[0, 1, 2]]), [0], 32, 1).any()
    # a prompt's last row is the decode of that length
    qs = rng.standard_normal((7, 1, 128)).astype(np.float32)
    pre = OP.sdpa_int4_paged_prefill(qs, pages, [0, 1, 2], 60, 32, 1, window=9, sinks=3)
    for i in range(7):
        one = OP.sdpa_int4_paged(qs[i][None], pages, np.array([[0, 1, 2]]), [61 + i], 32, 1, window=9, sinks=3)
        np.testing.assert_allclose(pre[i], one[0], atol=1e-12)


def test_oracle_pool_operations():
    page = np.arange(8, dtype=np.int32).reshape(1, 8, 1)
    p = OP.Pool(np.full((4, 3), -1, np.int32), np.zeros(8, np.int32), np.zeros(4, np.int32), 32, [page])
    assert list(p.reserve([40, 0, 32, 97])) == [1, 0, 1, 0]  # 97 rows exceed three pages
    assert p.tables.tolist() == [[0, 1, -1], [-1] * 3, [2, -1, -1], [-1] * 3]
    p.lengths[:] = [40, 0, 32, 0]
    assert list(p.fork([-1, 0, -1, 2])) == [0, 1, 0, 1]
    assert p.tables[1].tolist() == [0, 3, -1] and p.tables[3].tolist() == [2, -1, -1]
    assert p.refs.tolist() == [2, 1, 2, 1, 0, 0, 0, 0] and p.pages[0][0, 3, 0] == 1
    assert list(p.fork([-1, 0, -1, -1])) == [0] * 4  # not empty
    p.free([1, 0, 0, 0])
    assert p.refs.tolist() == [1, 0, 2, 1, 0, 0, 0, 0] and p.tables[0].tolist() == [-1] * 3
    assert p.compact() == 3
    assert p.tables.tolist() == [[-1] * 3, [0, 1, -1], [2, -1, -1], [2, -1, -1]]
    assert p.refs.tolist() == [1, 1, 2] + [0] * 5 and p.pages[0][0, 1, 0] == 1
    p.lengths[1] = 90
    p.evict(20, 0)
    assert p.tables[1].tolist() == [-1, -1, -1] and p.refs.tolist() == [0, 0, 2] + [0] * 5
    assert list(p.reserve([300, 6, 64, 0])) == [0, 1, 1, 0]
