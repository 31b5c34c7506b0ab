"""The operators of the paged int4 KV cache: appending to it, attending it
(single tokens, batches that share a prefix, prompts; each with a sliding
window and first tokens that stay visible), and moving its pages.

A cache is a pool of pages, tensors [pages, Hkv, page, .] in the library's
int4 layout, and a table of page numbers per sequence.  Shapes are those of the
other benchmarks: Hq 32 / Hkv 16 / D 256 (sliding layers), Hq 32 / Hkv 4 / D 512
(global layers), D 128 (the small configurations).  Queries and keys are
RMS-normed N(0, 1) per head vector and are scored with scale 1; values are
N(0, 1).

With ``own`` false an operator is computed by elementary torch operations in
32 bits, else by the library's calls.
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the first tokens of one small chat: nothing but latency
        dict(name="decode_tiny", kind="attend", Hq=2, Hkv=1, D=128, B=1, lo=33, hi=33, shared=0, page=32, window=0,
             sinks=0, q="f32", sb="f32"),
        # a sliding layer of a serving batch that keeps the first four tokens
        # in sight
        dict(name="decode_sinks", kind="attend", Hq=32, Hkv=16, D=256, B=32, lo=512, hi=8192, shared=0, page=64,
             window=1024, sinks=4, q="bf16", sb="f16"),
        # a full-attention layer of a large batch of unequal lengths
        dict(name="decode_ragged", kind="attend", Hq=32, Hkv=16, D=256, B=64, lo=512, hi=16384, shared=0, page=64,
             window=0, sinks=0, q="bf16", sb="f16"),
        # a global layer of a few long sequences
        dict(name="decode_global", kind="attend", Hq=32, Hkv=4, D=512, B=8, lo=1024, hi=32768, shared=0, page=128,
             window=0, sinks=0, q="f16", sb="f16"),
        # four samples of one prompt, a few tokens in
        dict(name="prefix_samples", kind="attend", Hq=16, Hkv=8, D=128, B=4, lo=1, hi=100, shared=1024, page=32,
             window=0, sinks=0, q="f32", sb="f32"),
        # many questions about one long document
        dict(name="prefix_document", kind="attend", Hq=32, Hkv=16, D=256, B=64, lo=1, hi=512, shared=32768, page=64,
             window=0, sinks=0, q="bf16", sb="f16"),
        # a short chunk of a prompt behind a longer context, sliding layer
        dict(name="prompt_chunk", kind="prompt", Hq=32, Hkv=16, D=256, prior=4001, new=67, page=64, window=1024,
             sinks=4, q="f16", sb="f16"),
        # a long chunk through a global layer
        dict(name="prompt_long", kind="prompt", Hq=32, Hkv=4, D=512, prior=6144, new=2048, page=128, window=0,
             sinks=0, q="bf16", sb="f16"),
        # one token of every sequence into the cache
        dict(name="append_step", kind="append", Hkv=8, D=128, B=64, new=1, lo=1, hi=31, page=32, x="bf16", sb="f16"),
        # the rows of two prompts
        dict(name="append_prompt", kind="append", Hkv=16, D=256, B=2, new=2048, lo=0, hi=100, page=64, x="bf16",
             sb="f16"),
        # eight prompts, each continued seven ways: the children of the last
        # round end, the next ones share their parents' pages
        dict(name="pages_fork", kind="fork", layers=8, Hkv=16, D=256, parents=8, children=56, lo=700, hi=2000,
             page=64, sb="f16"),
        # a pool that half its sequences have left, to be packed
        dict(name="pages_compact", kind="compact", layers=4, Hkv=16, D=256, B=48, lo=100, hi=2000, page=64,
             sb="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "prefix", "prefix", "prompt", "prompt", "append", "fork",
                       "compact"])
    q = rng.choice(["bf16", "bf16", "f16", "f32"])
    sb = rng.choice(["f16", "f16", "f32"])
    Hq, Hkv, D = rng.choice([(32, 16, 256), (32, 16, 256), (32, 4, 512), (16, 8, 128), (32, 8, 128), (8, 1, 256)])
    page = rng.choice([32, 64, 64, 128, 256])
    window = rng.choice([0, 0, _log(rng, 100, 2000)])
    sinks = rng.choice([0, 4, rng.randint(1, 70)]) if window else 0
    if kind in ("decode", "prefix"):
        shared = 0 if kind == "decode" else max(1, _log(rng, 256, 16384) // page) * page
        hi = _log(rng, 64, 8192 if kind == "decode" else 512)
        return dict(kind="attend", Hq=Hq, Hkv=Hkv, D=D, B=_log(rng, 1, 48), lo=max(1, hi // rng.choice([1, 4, 16])),
                    hi=hi, shared=shared, page=page, window=window, sinks=sinks, q=q, sb=sb)
    if kind == "prompt":
        return dict(kind=kind, Hq=Hq, Hkv=Hkv, D=D, prior=rng.choice([0, _log(rng, 16, 6000)]), new=_log(rng, 2, 1024),
                    page=page, window=window, sinks=sinks, q=q, sb=sb)
    if kind == "append":
        B = _log(rng, 1, 64)
        return dict(kind=kind, Hkv=Hkv, D=D, B=B, new=_log(rng, 1, max(2, 2048 // B)), lo=0, hi=rng.randint(1, 200),
                    page=page, x=q, sb=sb)
    if kind == "fork":
        parents = rng.randint(1, 8)
        return dict(kind=kind, layers=rng.randint(1, 8), Hkv=Hkv, D=D, parents=parents,
                    children=parents * rng.randint(1, 7), lo=1, hi=_log(rng, 60, 2000), page=min(page, 128), sb=sb)
    return dict(kind=kind, layers=rng.randint(1, 4), Hkv=Hkv, D=D, B=rng.randint(2, 48), lo=1, hi=_log(rng, 60, 2000),
                page=min(page, 128), sb=sb)


def _lens(lo, hi, n):
    """n lengths spread over lo .. hi."""
    return [lo + int((hi - lo + 1) * (i * 0.6180339887498949 % 1.0)) for i in range(n)]


def _pages(n, page):
    return -(-n // page)


def _visible(n, window, sinks, first=0):
    """Keys of first .. n - 1 that the query at n - 1 attends."""
    lo = max(n - window, first) if window else first
    return max(0, n - lo) + max(0, min(sinks, lo) - first)


def _attend_lens(case):
    return [case["shared"] + n for n in _lens(case["lo"], case["hi"], case["B"])]


def work(case):
    kind = case["kind"]
    if kind == "append":
        vals = 2 * case["B"] * case["new"] * case["Hkv"] * case["D"]
        # and the pool's values, which the pass hands back
        rows = sum(_pages(n + case["new"], case["page"]) for n in _lens(case["lo"], case["hi"], case["B"])) * case["page"]
        back = 2 * rows * case["Hkv"] * case["D"]
        return {"bytes": vals * (_SIZE[case["x"]] + 0.5 + _SIZE[case["sb"]] / 32) + back * (4.5 + _SIZE[case["sb"]] / 32),
                "flops": 8 * vals + 2 * back}
    if kind in ("fork", "compact"):
        page = 2 * case["layers"] * case["Hkv"] * case["page"] * case["D"] * (0.5 + _SIZE[case["sb"]] / 32)
        if kind == "fork":
            lens = _lens(case["lo"], case["hi"], case["parents"])
            kids = [lens[i % case["parents"]] for i in range(case["children"])]
            copies = sum(n % case["page"] > 0 for n in kids)
            entries = sum(_pages(n, case["page"]) for n in kids)
            return {"bytes": 2 * copies * page + 16 * entries, "flops": entries}
        lens = _lens(case["lo"], case["hi"], case["B"])
        used = [_pages(n, case["page"]) for n in lens]
        live, total = sum(used[::2]), sum(used)
        # of pages that lie anywhere, this share is behind the first `live`
        return {"bytes": 2 * live * (1 - live / total) * page + 8 * total + 8 * sum(used[::2]), "flops": total}
    row = case["Hkv"] * case["D"] * (1 + _SIZE[case["sb"]] / 16)  # one token's K and V
    if kind == "attend":
        P, lens = case["shared"], _attend_lens(case)
        suffix = sum(_visible(n, case["window"], case["sinks"], P) for n in lens)
        every = sum(_visible(n, case["window"], case["sinks"]) for n in lens)
        prefix = 0
        if P:  # keys of the prefix that any sequence attends
            lo = min(max(0, n - case["window"]) if case["window"] else 0 for n in lens)
            prefix = max(0, P - lo) + min(case["sinks"], lo, P)
        return {"bytes": (prefix + suffix) * row + len(lens) * case["Hq"] * case["D"] * (4 + _SIZE[case["q"]]),
                "flops": 4 * case["Hq"] * case["D"] * every}
    prior, new = case["prior"], case["new"]
    every = sum(_visible(prior + i + 1, case["window"], case["sinks"]) for i in range(new))
    lo = max(0, prior + 1 - case["window"]) if case["window"] else 0
    keys = prior + new - lo + min(case["sinks"], lo)
    return {"bytes": keys * row + new * case["Hq"] * case["D"] * (4 + _SIZE[case["q"]]),
            "flops": 4 * case["Hq"] * case["D"] * every}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _quantize(x, sb):
    """The cache's number format (MLX affine int4, groups of 64), decided in
    32 bits: words [.., D/8] int32, scale and bias [.., D/64].  A quotient of
    64 bits rounded to 32 is the correctly rounded one of 32; many groups of
    16-bit inputs have their edge at 7.5 steps, where the next one differs."""
    def div(a, b):
        return (a.double() / b).float()
    g = x.float().reshape(*x.shape[:-1], -1, 64)
    mx, mn = g.amax(-1), g.amin(-1)
    scale = div(mx - mn, 15.0).clamp(min=1e-7)
    side = mn.abs() > mx.abs()
    scale = torch.where(side, scale, -scale)
    edge = torch.where(side, mn, mx)
    q0 = torch.round(div(edge, scale.double()))
    scale = torch.where(q0 != 0, div(edge, q0.double()), scale)
    bias = torch.where(q0 != 0, edge, torch.zeros_like(edge))
    n = torch.round(div(g - bias[..., None], scale[..., None].double())).clamp(0, 15).to(torch.int32)
    sh = torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)
    words = (n.reshape(*x.shape[:-1], -1, 8) << sh).sum(-1, dtype=torch.int32)
    return words, scale.to(sb), bias.to(sb)


def _values(w, s, b):
    """The values that packed rows stand for, in 32 bits."""
    sh = torch.arange(0, 32, 4, device=w.device, dtype=torch.int32)
    n = ((w.view(torch.int32)[..., None] >> sh) & 15).reshape(*s.shape, 64).float()
    return (n * s.float()[..., None] + b.float()[..., None]).flatten(-2)


def _rms(x):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)


def _pool(g, lead, D, sb):
    """Page tensors (K words, scales, biases, then V's) of shape lead + (.,),
    rows drawn from a bank of quantized ones."""
    rows, out = math.prod(lead), []
    for norm in (True, False):
        x = torch.randn((16384, D), generator=g, device="cuda")
        bank = _quantize(_rms(x) if norm else x, sb)
        at = torch.randint(0, 16384, (rows,), generator=g, device="cuda")
        out += [t[at].reshape(*lead, t.shape[-1]) for t in bank]
    return [t.view(torch.uint32) if t.dtype == torch.int32 else t for t in out]


def _table(g, used, total, width):
    """Tables of sequences of used[i] pages, in any order of the pool."""
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    t = torch.full((len(used), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(used):
        t[i, :n] = order[at:at + n]
        at += n
    return t


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, kind, s = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17), case["kind"], dict(case)
    page, D, sb = case["page"], case["D"], _DT[case["sb"]]
    if kind == "attend":
        lens, pre = _attend_lens(case), case["shared"] // page
        used = [_pages(n, page) - pre for n in lens]
        total = pre + sum(used)
        s["tables"] = _table(g, [pre] + used, total, pre + max(used))
        # every sequence's table starts with the shared pages
        own_pages = s["tables"][1:, :max(used)]
        s["tables"] = torch.cat([s["tables"][:1, :pre].expand(len(lens), -1), own_pages], 1).contiguous()
        s["lens"], s["longest"] = _ints(lens), max(lens)
        s["pages"] = _pool(g, (total, case["Hkv"], page), D, sb)
        s["q_"] = _rms(torch.randn((case["B"], case["Hq"], D), generator=g, device="cuda")).to(_DT[case["q"]])
    elif kind == "prompt":
        total = _pages(case["prior"] + case["new"], page)
        s["tables"] = _table(g, [total], total, total)[0].contiguous()
        s["pages"] = _pool(g, (total, case["Hkv"], page), D, sb)
        s["q_"] = _rms(torch.randn((case["new"], case["Hq"], D), generator=g, device="cuda")).to(_DT[case["q"]])
    elif kind == "append":
        lens = _lens(case["lo"], case["hi"], case["B"])
        used = [_pages(n + case["new"], page) for n in lens]
        s["tables"] = _table(g, used, sum(used), max(used))
        s["lens"] = _ints(lens)
        s["pages"] = _pool(g, (sum(used), case["Hkv"], page), D, sb)
        x = torch.randn((2, case["B"], case["Hkv"], case["new"], D), generator=g, device="cuda")
        s["k"], s["v"] = _rms(x[0]).to(_DT[case["x"]]), x[1].to(_DT[case["x"]])
    elif kind == "fork":
        lens = _lens(case["lo"], case["hi"], case["parents"])
        used = [_pages(n, page) for n in lens]
        total = sum(used) + case["children"] + 3
        kids = torch.zeros((case["children"], max(used)), dtype=torch.int32, device="cuda") - 1
        s["tables"] = torch.cat([_table(g, used, total, max(used)), kids])
        s["refs"] = torch.zeros(total, dtype=torch.int32, device="cuda")
        s["refs"][s["tables"][s["tables"] >= 0].long()] = 1
        s["lens"] = _ints(lens + [0] * case["children"])
        s["parents_of"] = _ints([-1] * case["parents"] + [i % case["parents"] for i in range(case["children"])])
        s["ended"] = (s["parents_of"] >= 0).int()
        s["pages"] = _pool(g, (case["layers"], total, case["Hkv"], page), D, sb)
    else:
        used = [_pages(n, page) for n in _lens(case["lo"], case["hi"], case["B"])]
        s["tables"] = _table(g, used, sum(used), max(used))
        s["tables"][1::2] = -1  # these sequences have ended
        s["refs"] = torch.zeros(sum(used), dtype=torch.int32, device="cuda")
        s["refs"][s["tables"][s["tables"] >= 0].long()] = 1
        s["pages"] = _pool(g, (case["layers"], sum(used), case["Hkv"], page), D, sb)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _softmax_product(parts):
    """softmax over the parts' scores (masked ones -inf) times their values;
    rows that attend nothing give 0."""
    m = torch.stack([sc.amax(-1) for sc, _ in parts]).amax(0)[..., None]
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = [torch.exp(sc - m) for sc, _ in parts]
    total = sum(x.sum(-1, keepdim=True) for x in e)
    out = sum(torch.matmul(x, v) for x, (_, v) in zip(e, parts))
    return torch.where(total > 0, out / total, torch.zeros_like(out))


def _seen(t, n, window, sinks):
    """Whether the query at n - 1 attends key t."""
    ok = t < n
    return ok & ((t < sinks) | (t >= n - window)) if window else ok


def _gathered(pool, table):
    """Values [.., Hkv, rows, D] of the pages of tables [.., n]."""
    at = table.clamp(min=0).long()
    x = _values(*(t[at] for t in pool)).movedim(-4, -3)  # [.., Hkv, n, page, D]
    return x.flatten(-3, -2)


def _attend_plain(s):
    B, Hq, D = s["q_"].shape
    Hkv, page, P = s["Hkv"], s["page"], s["shared"]
    K, V = ([t.view(torch.int32) if t.dtype == torch.uint32 else t for t in s["pages"][i:i + 3]] for i in (0, 3))
    q = s["q_"].float().reshape(B, Hkv, Hq // Hkv, D)
    n = s["lens"][:, None, None, None]
    tail = s["tables"][:, P // page:]
    k, v = _gathered(K, tail), _gathered(V, tail)
    t = P + torch.arange(k.shape[-2], device="cuda")
    sc = torch.matmul(q, k.transpose(-1, -2))
    parts = [(sc.masked_fill(~_seen(t, n, s["window"], s["sinks"]), -math.inf), v)]
    if P:
        head = s["tables"][0, :P // page]
        k, v = _gathered(K, head), _gathered(V, head)  # [Hkv, P, D]
        rows = q.transpose(0, 1).reshape(Hkv, -1, D)
        sc = torch.matmul(rows, k.transpose(-1, -2)).reshape(Hkv, B, -1, P).transpose(0, 1)
        sc = sc.masked_fill(~_seen(torch.arange(P, device="cuda"), n, s["window"], s["sinks"]), -math.inf)
        parts.append((sc, v))
    return _softmax_product(parts).reshape(B, Hq, D)


def _prompt_plain(s):
    new, Hq, D = s["q_"].shape
    Hkv, L = s["Hkv"], s["prior"] + new
    K, V = ([t.view(torch.int32) if t.dtype == torch.uint32 else t for t in s["pages"][i:i + 3]] for i in (0, 3))
    k, v = _gathered(K, s["tables"]), _gathered(V, s["tables"])
    q = s["q_"].float().reshape(new, Hkv, -1, D).permute(1, 2, 0, 3)  # [Hkv, heads, new, D]
    n = s["prior"] + 1 + torch.arange(new, device="cuda")[:, None]
    sc = torch.matmul(q, k[:, None].transpose(-1, -2))
    sc = sc.masked_fill(~_seen(torch.arange(k.shape[-2], device="cuda"), n, s["window"], s["sinks"]), -math.inf)
    return _softmax_product([(sc, v[:, None])]).permute(2, 0, 1, 3).reshape(new, Hq, D)


def _append_plain(s):
    B, Hkv, T, D = s["k"].shape
    at = s["lens"].long()[:, None] + torch.arange(T, device="cuda")  # [B, T]
    to = torch.gather(s["tables"].long(), 1, at // s["page"])
    new = _quantize(s["k"], s["pages"][1].dtype) + _quantize(s["v"], s["pages"][1].dtype)
    pages = [t.view(torch.int32) if t.dtype == torch.uint32 else t for t in s["pages"]]
    for pool, x in zip(pages, new):
        pool[to, :, at % s["page"]] = x.transpose(1, 2)
    return _values(*pages[:3]), _values(*pages[3:])


def _free_plain(tables, refs, lens, which):
    rows = which[:, None] != 0
    gone = (tables >= 0) & rows
    refs.index_add_(0, tables.clamp(min=0).flatten().long(), -gone.flatten().int())
    tables.masked_fill_(rows, -1)
    lens.masked_fill_(which != 0, 0)


def _fork_plain(s):
    """The children's tables: their parents' full pages, shared, and a copy of
    the page that is not full; copies go to the lowest free pages."""
    tables, refs, lens, page = s["tables"], s["refs"], s["lens"], s["page"]
    _free_plain(tables, refs, lens, s["ended"])
    par = s["parents_of"].clamp(min=0).long()
    kid = s["parents_of"] >= 0
    n = torch.where(kid, lens[par], torch.zeros_like(lens))
    part = kid & (n % page > 0)
    before = torch.cumsum(part, 0) - part.long()
    free = torch.nonzero(refs <= 0).flatten()
    granted = kid & (~part | (before < free.numel()))
    part &= granted
    dst = free[before[part]]
    src = tables[par][part].gather(1, (n[part] // page)[:, None].long()).flatten().long()
    e = torch.arange(tables.shape[1], device="cuda")
    full = granted[:, None] & (e < (n // page)[:, None])
    shared = torch.where(full, tables[par], torch.full_like(tables, -1))
    refs.index_add_(0, shared.clamp(min=0).flatten().long(), (shared >= 0).flatten().int())
    refs[dst] = 1
    tables.copy_(torch.where(granted[:, None], shared, tables))
    tables[part, (n[part] // page).long()] = dst.int()
    lens.copy_(torch.where(granted, n, lens))
    pages = [t.view(torch.int32) if t.dtype == torch.uint32 else t for t in s["pages"]]
    for t in pages:
        t[:, dst] = t[:, src]
    return dict(tables=tables, refs=refs, lengths=lens, granted=granted.int(), pages=pages)


def _compact_plain(s):
    """The pages in use to the front: the k-th free place there takes the k-th
    page from behind."""
    tables, refs = s["tables"], s["refs"]
    live = refs > 0
    n = live.sum()
    at = torch.arange(refs.numel(), device="cuda")
    hole, mover = torch.nonzero(~live & (at < n)).flatten(), torch.nonzero(live & (at >= n)).flatten()
    to = at.clone()
    to[mover] = hole
    new = torch.where(tables >= 0, to[tables.clamp(min=0).long()].int(), tables)
    out = torch.where(live & (at < n), refs, torch.zeros_like(refs))
    out[hole] = refs[mover]
    pages = [t.view(torch.int32) if t.dtype == torch.uint32 else t for t in s["pages"]]
    for t in pages:
        t[:, hole] = t[:, mover]
    return dict(tables=new, refs=out, live=n.int(), pages=pages)


def _words(pages):
    return [t.view(torch.int32) if t.dtype == torch.uint32 else t for t in pages]


def _own(s):
    from gemma4metal_amd import paged, turboquant as tq
    kind, pages = s["kind"], s["pages"]
    if kind == "attend":
        return paged.sdpa_int4_paged(s["q_"], *pages, s["tables"], s["lens"], s["Hq"] // s["Hkv"], 1.0, s["window"],
                                     s["sinks"], shared_prefix=s["shared"], max_kv_len=s["longest"])
    if kind == "prompt":
        return paged.sdpa_int4_paged_prefill(s["q_"], *pages, s["tables"], s["prior"], s["Hq"] // s["Hkv"], 1.0,
                                             s["window"], s["sinks"])
    if kind == "append":
        paged.kv_append_int4_paged(s["k"], s["v"], *pages, s["tables"], s["lens"])
        return tq.dequantize(*pages[:3]), tq.dequantize(*pages[3:])
    if kind == "fork":
        paged.kv_pages_free(s["tables"], s["refs"], s["lens"], s["ended"])
        granted = paged.kv_pages_fork(pages, s["tables"], s["refs"], s["lens"], s["parents_of"])
        return dict(tables=s["tables"], refs=s["refs"], lengths=s["lens"], granted=granted, pages=_words(pages))
    tables, refs, live = paged.kv_pages_compact(pages, s["tables"], s["refs"])
    return dict(tables=tables, refs=refs, live=live, pages=_words(pages))


def run(state):
    if own:
        return _own(state)
    return {"attend": _attend_plain, "prompt": _prompt_plain, "append": _append_plain, "fork": _fork_plain,
            "compact": _compact_plain}[state["kind"]](state)


# ---------------------------------------------------------------------------
# the definition
# ---------------------------------------------------------------------------

def _rows64(pool, pages, h, n):
    """The first n rows of head h over a list of pages, in 64 bits."""
    w, s, b = (t[pages, h].flatten(0, 1)[:n] for t in pool)
    w = w.view(torch.int32).long() & 0xFFFFFFFF
    nib = torch.stack([(w >> (4 * i)) & 15 for i in range(8)], -1).reshape(n, -1, 64).double()
    return torch.addcmul(b.double()[..., None], nib, s.double()[..., None]).reshape(n, -1)


def _row64(scores, keep, v):
    """One softmax row set; scores [rows, n], keep [rows, n] or [n]."""
    scores = scores.masked_fill(~keep, -math.inf)
    return torch.nan_to_num(torch.softmax(scores, -1), nan=0.0) @ v


def _exact_attention(case, s):
    Hkv, G, W, sinks = case["Hkv"], case["Hq"] // case["Hkv"], case["window"], case["sinks"]
    pool = [t.view(torch.int32) if t.dtype == torch.uint32 else t for t in s["pages"]]
    q, lens = s["q_"].double(), s["lens"].tolist() if "lens" in s else None
    out = torch.zeros_like(q)
    for h in range(Hkv):
        head = slice(h * G, h * G + G)
        if case["kind"] == "prompt":
            n = case["prior"] + case["new"]
            k, v = (_rows64(pool[i:i + 3], s["tables"].long(), h, n) for i in (0, 3))
            pos = case["prior"] + torch.arange(case["new"], device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            keep = (j <= pos) & ((pos - j < W) | (j < sinks) if W else True)
            for i in range(h * G, h * G + G):
                out[:, i] = _row64(q[:, i] @ k.t(), keep, v)
            continue
        P = case["shared"]
        if P:
            pre = [_rows64(pool[i:i + 3], s["tables"][0, :P // case["page"]].long(), h, P) for i in (0, 3)]
        for b in range(case["B"]):
            n = lens[b]
            mine = s["tables"][b, P // case["page"]:_pages(n, case["page"])].long()
            kv = [_rows64(pool[i:i + 3], mine, h, n - P) for i in (0, 3)]
            k, v = (torch.cat([x, y]) for x, y in zip(pre, kv)) if P else kv
            j = torch.arange(n, device="cuda")
            keep = (n - 1 - j < W) | (j < sinks) if W else j < n
            out[b, head] = _row64(q[b, head] @ k.t(), keep, v)
    return out


def _nibbles32(x):
    """The quantization rule as it is defined, in steps of 32 bits: the values
    that rows x stand for, as functions of the stored scale's type."""
    x = x.float().cpu().numpy().reshape(-1, 64)
    f = np.float32
    hi, lo = x.max(1), x.min(1)
    step = np.maximum((hi - lo) / f(15), f(1e-7))
    down = np.abs(lo) > np.abs(hi)
    step = np.where(down, step, -step)
    edge = np.where(down, lo, hi)
    near = np.rint(edge / step)
    fits = near != 0
    step = np.where(fits, edge / np.where(fits, near, f(1)), step)
    start = np.where(fits, edge, f(0))
    return np.clip(np.rint((x - start[:, None]) / step[:, None]), 0, 15), step, start


def _exact_append(case, s):
    out = []
    sb = np.float16 if case["sb"] == "f16" else np.float32
    page, T, D = case["page"], case["new"], case["D"]
    for first, x in ((0, s["k"]), (3, s["v"])):
        pool = [t.view(torch.int32) if t.dtype == torch.uint32 else t for t in s["pages"][first:first + 3]]
        N, Hkv = pool[0].shape[:2]
        vals = torch.stack([_rows64(pool, torch.arange(N, device="cuda"), h, N * page).reshape(N, page, D)
                            for h in range(Hkv)], 1)
        nib, step, start = _nibbles32(x)
        new = nib.astype(np.float64) * step.astype(sb).astype(np.float64)[:, None] + start.astype(sb).astype(np.float64)[:, None]
        new = torch.from_numpy(new).cuda().reshape(x.shape)
        for b in range(case["B"]):
            n = int(s["lens"][b])
            for e in range(n // page, _pages(n + T, page)):
                a, z = max(n, e * page), min(n + T, (e + 1) * page)
                vals[int(s["tables"][b, e]), :, a - e * page:z - e * page] = new[b, :, a - n:z - n]
        out.append(vals)
    return tuple(out)


def _exact_fork(case, s):
    tables, refs, lens = s["tables"].tolist(), s["refs"].tolist(), s["lens"].tolist()
    parents, page, copies = s["parents_of"].tolist(), case["page"], []
    granted = [0] * len(parents)
    spare = iter([p for p, r in enumerate(refs) if r <= 0])
    for row, par in enumerate(parents):
        if par < 0:
            continue
        full, rest = divmod(lens[par], page)
        if rest:
            dst = next(spare, None)
            if dst is None:
                continue
            copies.append((tables[par][full], dst))
            refs[dst] = 1
            tables[row][full] = dst
        for e in range(full):
            tables[row][e] = tables[par][e]
            refs[tables[par][e]] += 1
        lens[row], granted[row] = lens[par], 1
    pages = [t.view(torch.int32) if t.dtype == torch.uint32 else t for t in s["pages"]]
    for src, dst in copies:
        for t in pages:
            t[:, dst] = t[:, src]
    return dict(tables=_ints(tables), refs=_ints(refs), lengths=_ints(lens), granted=_ints(granted), pages=pages)


def _exact_compact(case, s):
    refs = s["refs"].tolist()
    live = [p for p, r in enumerate(refs) if r > 0]
    n, keep = len(live), set(live)
    to = dict(zip([p for p in live if p >= n], [p for p in range(n) if p not in keep]))
    pages = [t.view(torch.int32) if t.dtype == torch.uint32 else t for t in s["pages"]]
    for src, dst in to.items():
        for t in pages:
            t[:, dst] = t[:, src]
    out = [0] * len(refs)
    for p in live:
        out[to.get(p, p)] = refs[p]
    tables = [[to.get(p, p) for p in row] for row in s["tables"].tolist()]
    return dict(tables=_ints(tables), refs=_ints(out), live=torch.tensor(n, dtype=torch.int32), pages=pages)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("attend", "prompt"):
        return _exact_attention(case, s)
    return {"append": _exact_append, "fork": _exact_fork, "compact": _exact_compact}[kind](case, s)
