"""The operators of beam search and of batched prompts over the int4 KV cache:
choosing the next beams from the logits, reordering the cached sequences by the
beams chosen (pages, and contiguous caches), and attention of a chunk of new
tokens of every sequence of a batch over its pages.

Head shapes are those of the other benchmarks: Hq 32 / Hkv 16 / D 256 (sliding
layers), Hq 32 / Hkv 4 / D 512 (global layers), D 128 (the small
configurations).  Queries and keys are RMS-normed N(0, 1) per head vector and are
scored with scale 1; values are N(0, 1); logits are N(0, 3) with a few tokens that
stand out.

With ``own`` false an operator is computed by elementary torch operations in 32
bits (log-probabilities in 64: beams are told apart by their sums), else by the
library's calls.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one request with four beams and a small vocabulary: latency
        dict(name="select_small", kind="select", B=1, W=4, V=32000, K=4, x="f32", ended=0),
        # a batch with an odd vocabulary, twice as many candidates as beams, some
        # beams at their end
        dict(name="select_odd", kind="select", B=8, W=5, V=50257, K=10, x="f16", ended=3),
        # a large batch with a large vocabulary
        dict(name="select_large", kind="select", B=32, W=8, V=262144, K=8, x="bf16", ended=8),
        # one request's beams, a single layer: latency
        dict(name="pages_small", kind="pages", layers=1, Hkv=8, D=128, groups=1, W=4, dropped=1, prompt=100, lo=1,
             hi=20, page=32, sb="f32"),
        # the beams of eight requests behind their prompts, eight layers
        dict(name="pages_beams", kind="pages", layers=8, Hkv=16, D=256, groups=8, W=8, dropped=3, prompt=1000, lo=10,
             hi=250, page=64, sb="f16"),
        # one request's beams in a contiguous cache, just begun
        dict(name="cache_small", kind="cache", Hkv=8, D=128, groups=1, W=4, dropped=1, cap=128, lo=33, hi=33,
             sb="f32"),
        # the beams of eight requests in a contiguous cache
        dict(name="cache_beams", kind="cache", Hkv=16, D=256, groups=8, W=4, dropped=1, cap=4096, lo=700, hi=4000,
             sb="f16"),
        # two short chats, three new tokens each: latency
        dict(name="chunks_tiny", kind="chunks", Hq=2, Hkv=1, D=128, B=2, new=3, long=0, longs=0, lo=33, hi=60,
             page=32, window=0, sinks=0, q="f32", sb="f32"),
        # five proposed tokens of every sequence to be checked, a sliding layer
        dict(name="chunks_proposed", kind="chunks", Hq=32, Hkv=16, D=256, B=32, new=5, long=0, longs=0, lo=300,
             hi=6000, page=64, window=1024, sinks=4, q="bf16", sb="f16"),
        # a serving batch: most sequences one token, three of them chunks of prompts
        dict(name="chunks_mixed", kind="chunks", Hq=32, Hkv=8, D=128, B=24, new=1, long=201, longs=3, lo=100, hi=4000,
             page=64, window=0, sinks=0, q="f16", sb="f16"),
        # eight prompts at once, a sliding layer that still sees everything
        dict(name="chunks_prompts", kind="chunks", Hq=32, Hkv=16, D=256, B=8, new=300, long=700, longs=2, lo=0,
             hi=500, page=64, window=0, sinks=0, q="bf16", sb="f16"),
        # chunks of four long prompts, a global layer
        dict(name="chunks_global", kind="chunks", Hq=32, Hkv=4, D=512, B=4, new=500, long=0, longs=0, lo=1000,
             hi=8000, page=128, window=0, sinks=0, q="bf16", sb="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["select", "select", "pages", "cache", "chunks", "chunks", "chunks"])
    sb = rng.choice(["f16", "f16", "f32"])
    q = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "select":
        W, V = rng.randint(1, 12), _log(rng, 200, 262144)
        B = max(1, min(_log(rng, 1, 64), 32 * 262144 // (V * W)))
        K = rng.choice([W, W, 2 * W, rng.randint(1, 20)])
        return dict(kind=kind, B=B, W=W, V=V, K=K, x=q, ended=rng.choice([0, rng.randint(0, B * W - 1)]))
    W = rng.randint(2, 10)
    groups, dropped = _log(rng, 1, 8), rng.randint(0, W - 1)
    Hq, Hkv, D = rng.choice([(32, 16, 256), (32, 16, 256), (32, 4, 512), (16, 8, 128), (32, 8, 128), (8, 1, 256)])
    if kind == "pages":
        return dict(kind=kind, layers=rng.randint(1, 8), Hkv=Hkv, D=D, groups=groups, W=W, dropped=dropped,
                    prompt=_log(rng, 1, 1000), lo=1, hi=_log(rng, 2, 250), page=rng.choice([32, 64, 64, 128]), sb=sb)
    if kind == "cache":
        cap = _log(rng, 40, 32768 // W)
        return dict(kind=kind, Hkv=Hkv, D=D, groups=min(groups, max(1, 131072 // (cap * W))), W=W, dropped=dropped,
                    cap=cap, lo=1, hi=cap, sb=sb)
    new, longs = _log(rng, 1, 64), rng.choice([0, 0, rng.randint(1, 3)])
    window = rng.choice([0, 0, _log(rng, 100, 2000)])
    return dict(kind=kind, Hq=Hq, Hkv=Hkv, D=D, B=_log(rng, max(1, longs), 24), new=new,
                long=rng.randint(new, 260) if longs else 0, longs=longs, lo=rng.choice([0, 50]),
                hi=_log(rng, 60, 4000), page=rng.choice([32, 64, 64, 128, 256]), window=window,
                sinks=rng.choice([0, 4, rng.randint(1, 70)]) if window else 0, q=q, sb=sb)


def _lens(lo, hi, n):
    """n lengths spread over lo .. hi."""
    return [lo + int((hi - lo + 1) * (i * 0.6180339887498949 % 1.0)) for i in range(n)]


def _pages(n, page):
    return -(-n // page)


def _chunk_lens(case):
    """New tokens and lengths with them of a batch's sequences."""
    new = [case["long"] if i < case["longs"] else case["new"] for i in range(case["B"])]
    return new, [n + m for n, m in zip(new, _lens(case["lo"], case["hi"], case["B"]))]


def _visible(n, window, sinks):
    lo = max(n - window, 0) if window else 0
    return n - lo + min(sinks, lo)


def work(case):
    kind = case["kind"]
    if kind == "select":
        rows = case["B"] * case["W"] - case["ended"]
        n = rows * case["V"]
        return {"bytes": n * _SIZE[case["x"]] + 4 * case["B"] * (case["W"] + 3 * case["K"]), "flops": 4 * n}
    row = case["Hkv"] * case["D"] * (1 + _SIZE[case["sb"]] / 16)  # one token's K and V
    if kind == "pages":
        lens = [case["prompt"] + n for n in _lens(case["lo"], case["hi"], case["groups"])]
        copies = sum(case["dropped"] for n in lens if n % case["page"])
        entries = sum(case["W"] * _pages(n, case["page"]) for n in lens)
        return {"bytes": 2 * copies * case["layers"] * case["page"] * row + 8 * entries, "flops": entries}
    if kind == "cache":
        # every parent is read once; all beams but one change places, on average
        lens = _lens(case["lo"], case["hi"], case["groups"])
        kept = min(case["W"] - case["dropped"], case["W"] - 1)
        return {"bytes": sum(lens) * row * (kept + case["W"] - 1), "flops": 0}
    new, lens = _chunk_lens(case)
    W, every, keys = case["window"], 0, 0
    for n, L in zip(new, lens):
        every += sum(_visible(L - i, W, case["sinks"]) for i in range(n))
        lo = max(0, L - n + 1 - W) if W else 0
        keys += L - lo + min(case["sinks"], lo)
    return {"bytes": keys * row + sum(new) * case["Hq"] * case["D"] * (4 + _SIZE[case["q"]]),
            "flops": 4 * case["Hq"] * case["D"] * every}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _quantize(x, sb):
    """Rows in the cache's number format (affine int4, groups of 64): words
    [.., D/8] int32, scale and bias [.., D/64]."""
    g = x.float().reshape(*x.shape[:-1], -1, 64)
    mx, mn = g.amax(-1), g.amin(-1)
    scale = ((mx - mn) / 15).clamp(min=1e-7)
    n = torch.round((g - mn[..., None]) / scale[..., None]).clamp(0, 15).to(torch.int32)
    sh = torch.arange(0, 32, 4, device=x.device, dtype=torch.int32)
    words = (n.reshape(*x.shape[:-1], -1, 8) << sh).sum(-1, dtype=torch.int32)
    return words, scale.to(sb), mn.to(sb)


def _values(w, s, b):
    """The values that packed rows stand for, in 32 bits."""
    sh = torch.arange(0, 32, 4, device=w.device, dtype=torch.int32)
    n = ((w[..., None] >> sh) & 15).reshape(*s.shape, 64).float()
    return (n * s.float()[..., None] + b.float()[..., None]).flatten(-2)


def _rms(x):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)


def _pool(g, lead, D, sb):
    """Cache tensors (K words, scales, biases, then V's) of shape lead + (.,),
    rows drawn from a bank of quantized ones."""
    rows, out = math.prod(lead), []
    for norm in (True, False):
        x = torch.randn((16384, D), generator=g, device="cuda")
        bank = _quantize(_rms(x) if norm else x, sb)
        at = torch.randint(0, 16384, (rows,), generator=g, device="cuda")
        out += [t[at].reshape(*lead, t.shape[-1]) for t in bank]
    return [t.view(torch.uint32) if t.dtype == torch.int32 else t for t in out]


def _words(pages):
    return [t.view(torch.int32) if t.dtype == torch.uint32 else t for t in pages]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _parents(case, g):
    """Every beam's parent: of a group's W beams some are dropped, and others
    continued twice or more; in the order of their scores, which is any."""
    G, W = case["groups"], case["W"]
    kept = torch.rand((G, W), generator=g, device="cuda").argsort(1)[:, :W - case["dropped"]]
    more = torch.randint(0, kept.shape[1], (G, case["dropped"]), generator=g, device="cuda")
    every = torch.cat([kept, kept.gather(1, more)], 1)
    order = torch.rand((G, W), generator=g, device="cuda").argsort(1)
    return (every.gather(1, order) + W * torch.arange(G, device="cuda")[:, None]).flatten().int()


def prepare(case, seed):
    g, kind, s = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29), case["kind"], dict(case)
    if kind == "select":
        B, W, V = case["B"], case["W"], case["V"]
        x = 3 * torch.randn((B * W, V), generator=g, device="cuda")
        x.scatter_add_(1, torch.randint(0, V, (B * W, 8), generator=g, device="cuda"),
                       6 * torch.rand((B * W, 8), generator=g, device="cuda"))
        s["logits"] = x.reshape(B, W, V).to(_DT[case["x"]])
        s["scores"] = -30 - 10 * torch.rand((B, W), generator=g, device="cuda")
        s["finished"] = torch.zeros(B * W, dtype=torch.bool, device="cuda")
        s["finished"][torch.rand(B * W, generator=g, device="cuda").argsort()[:case["ended"]]] = True
        s["finished"] = s["finished"].reshape(B, W)
        return s
    D, sb = case["D"], _DT[case["sb"]]
    if kind == "pages":
        page, W, rows, at = case["page"], case["W"], [], 0
        lens = [case["prompt"] + n for n in _lens(case["lo"], case["hi"], case["groups"])]
        shared = case["prompt"] // page  # the prompt's full pages are every beam's
        for n in lens:
            head = list(range(at, at + shared))
            at += shared
            for _ in range(W):
                rows.append(head + list(range(at, at + _pages(n, page) - shared)))
                at += _pages(n, page) - shared
        total = at + 3
        order = torch.randperm(total, generator=g, device="cuda").int()
        width = max(len(r) for r in rows) + 1
        t = _ints([r + [-1] * (width - len(r)) for r in rows])
        s["tables"] = torch.where(t >= 0, order[t.clamp(min=0).long()], t)
        s["refs"] = torch.zeros(total, dtype=torch.int32, device="cuda")
        s["refs"].index_add_(0, s["tables"].clamp(min=0).flatten().long(), (s["tables"] >= 0).flatten().int())
        s["lens"] = _ints([n for n in lens for _ in range(W)])
        s["parents"] = _parents(case, g)
        s["pages"] = _pool(g, (case["layers"], total, case["Hkv"], page), D, sb)
    elif kind == "cache":
        lens = _lens(case["lo"], case["hi"], case["groups"])
        s["lens"] = _ints([n for n in lens for _ in range(case["W"])])
        s["parents"] = _parents(case, g)
        s["pages"] = _pool(g, (case["groups"] * case["W"], case["Hkv"], case["cap"]), D, sb)
    else:
        page, B = case["page"], case["B"]
        new, lens = _chunk_lens(case)
        used = [_pages(n, page) for n in lens]
        order = torch.randperm(sum(used), generator=g, device="cuda").int()
        t = torch.full((B, max(used)), -1, dtype=torch.int32, device="cuda")
        for i, n in enumerate(used):
            t[i, :n] = order[sum(used[:i]):sum(used[:i + 1])]
        s["tables"], s["lens"], s["longest"] = t, _ints(lens), max(lens)
        s["most"] = max(new)
        s["starts"] = _ints([sum(new[:i]) for i in range(B + 1)])
        s["pages"] = _pool(g, (sum(used), case["Hkv"], page), D, sb)
        s["q_"] = _rms(torch.randn((sum(new), case["Hq"], D), generator=g, device="cuda")).to(_DT[case["q"]])
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _select_plain(s):
    """The K candidates of a group with the largest sums of a beam's score and a
    token's log-probability, the lowest (beam, token) first among equals; a
    finished beam has one candidate, itself."""
    x = s["logits"].double()
    B, W, V = x.shape
    m = x.amax(-1, keepdim=True)
    lse = m + torch.exp(x - m).sum(-1, keepdim=True).log()
    total = s["scores"].double()[..., None] + (x - lse)
    ended = s["finished"][..., None]
    only = torch.where(torch.arange(V, device="cuda") == 0, s["scores"].double()[..., None], -math.inf)
    total = torch.where(ended, only, total).flatten(1)
    K, n = s["K"], W * V
    least = total.topk(min(K, n), 1).values[:, -1:]
    at = torch.arange(n, device="cuda", dtype=torch.float64)
    # those above the K-th value, and of its equals the first ones
    above = torch.where(total > least, total, -math.inf).topk(min(K, n), 1)
    equal = torch.where(total == least, -at, -math.inf).topk(min(K, n), 1)
    value = torch.cat([above.values, torch.where(equal.values > -math.inf, least, -math.inf)], 1)
    place = torch.cat([above.indices, equal.indices], 1)
    place = torch.where(value > -math.inf, place, n)
    by_place = place.argsort(dim=1, stable=True)
    value, place = value.gather(1, by_place), place.gather(1, by_place)
    best = value.argsort(dim=1, descending=True, stable=True)[:, :K]
    value, place = value.gather(1, best), place.gather(1, best)
    got = value > -math.inf
    parent = place // V + W * torch.arange(B, device="cuda")[:, None]
    return dict(scores=value.float(), parents=torch.where(got, parent, -1).int(),
                tokens=torch.where(got, place % V, -1).int())


def _pages_plain(s):
    """Every sequence becomes the continuation of its parent: its first child (the
    parent itself, where it is one) takes the parent's row over, the others share
    its full pages and get a copy of the last one, in the lowest free pages."""
    tables, refs, lens, page = s["tables"], s["refs"], s["lens"], s["page"]
    S, P = tables.shape
    par = s["parents"].long()
    me = torch.arange(S, device="cuda")
    first = torch.full((S,), S, device="cuda").scatter_reduce(0, par, torch.where(par == me, -1, me), "amin")
    heir = (par == me) | (first[par] == me)
    gone = (first == S)[:, None] & (tables >= 0)
    refs.index_add_(0, tables.clamp(min=0).flatten().long(), -gone.flatten().int())
    n, row = lens[par], tables[par]
    full = (n // page).long()
    last = row.gather(1, full.clamp(max=P - 1)[:, None]).flatten()
    part = ~heir & (n % page > 0) & (last >= 0)
    free = torch.nonzero(refs <= 0).flatten()
    before = torch.cumsum(part, 0) - part.long()
    ok = ~part | (before < free.numel())
    part &= ok
    dst, src = free[before[part]], last[part].long()
    e = torch.arange(P, device="cuda")
    share = (ok & ~heir)[:, None] & (e < full[:, None])
    shared = torch.where(share, row, torch.full_like(row, -1))
    refs.index_add_(0, shared.clamp(min=0).flatten().long(), (shared >= 0).flatten().int())
    refs[dst] = 1
    tables.copy_(torch.where(heir[:, None], row, shared))
    tables[part, full[part]] = dst.int()
    lens.copy_(torch.where(ok, n, torch.zeros_like(n)))
    pages = _words(s["pages"])
    for t in pages:
        t[:, dst] = t[:, src]
    return dict(tables=tables, refs=refs, lengths=lens, granted=ok.int(), pages=pages)


def _cache_plain(s):
    """Every sequence's rows become its parent's; those behind its length stay."""
    par, lens, pages = s["parents"].long(), s["lens"], _words(s["pages"])
    n = lens[par]
    taken = (torch.arange(s["cap"], device="cuda") < n[:, None])[:, None, :, None]
    for t in pages:
        t.copy_(torch.where(taken, t[par], t))
    lens.copy_(n)
    return dict(lengths=lens, pages=pages)


def _chunks_plain(s):
    """Attention of the packed queries, on sequences padded to the longest chunk."""
    starts, lens, T, page = s["starts"].long(), s["lens"].long(), s["most"], s["page"]
    Hkv, D = s["Hkv"], s["D"]
    new = starts[1:] - starts[:-1]
    i = torch.arange(T, device="cuda")
    real = i < new[:, None]  # [B, T]
    q = s["q_"].float()[(starts[:-1, None] + i).clamp(max=s["q_"].shape[0] - 1)]
    q = q.unflatten(2, (Hkv, -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, Hkv, heads x T, D]
    at = s["tables"].clamp(min=0).long()
    k, v = (_values(*(t[at] for t in _words(s["pages"][x:x + 3]))).movedim(2, 1).flatten(2, 3) for x in (0, 3))
    t = torch.arange(k.shape[2], device="cuda")
    n = (lens - new)[:, None] + i + 1  # [B, T]: keys up to the query's own
    keep = t < n[..., None]
    if s["window"]:
        keep &= (t < s["sinks"]) | (t >= n[..., None] - s["window"])
    sc = torch.matmul(q, k.transpose(-1, -2)).unflatten(2, (-1, T))
    sc = sc.masked_fill(~keep[:, None, None], -math.inf).flatten(2, 3)
    e = torch.exp(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    o = o.unflatten(2, (-1, T)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, T, Hq, D]
    return o[real]


def _own(s):
    from gemma4metal_amd import beam, paged, turboquant as tq
    kind = s["kind"]
    if kind == "select":
        scores, parents, tokens = beam.beam_select(s["logits"], s["scores"], s["K"], finished=s["finished"])
        return dict(scores=scores, parents=parents, tokens=tokens)
    pages = s["pages"]
    if kind == "pages":
        granted = paged.kv_pages_reorder(pages, s["tables"], s["refs"], s["lens"], s["parents"])
        return dict(tables=s["tables"], refs=s["refs"], lengths=s["lens"], granted=granted, pages=_words(pages))
    if kind == "cache":
        tq.kv_reorder_int4(*pages, s["lens"], s["parents"])
        return dict(lengths=s["lens"], pages=_words(pages))
    return paged.sdpa_int4_paged_chunks(s["q_"], *pages, s["tables"], s["starts"], s["lens"], s["Hq"] // s["Hkv"], 1.0,
                                        s["window"], s["sinks"], max_new=s["most"], max_kv_len=s["longest"])


def run(state):
    if own:
        return _own(state)
    return {"select": _select_plain, "pages": _pages_plain, "cache": _cache_plain,
            "chunks": _chunks_plain}[state["kind"]](state)


# ---------------------------------------------------------------------------
# the definition
# ---------------------------------------------------------------------------

def _exact_select(case, s):
    B, W, V = s["logits"].shape
    out = dict(scores=torch.full((B, case["K"]), -math.inf, dtype=torch.float64, device="cuda"),
               parents=_ints([[-1] * case["K"]] * B), tokens=_ints([[-1] * case["K"]] * B))
    for b in range(B):
        rows = torch.log_softmax(s["logits"][b].double(), -1) + s["scores"][b].double()[:, None]
        for w in torch.nonzero(s["finished"][b]).flatten().tolist():
            rows[w] = -math.inf
            rows[w, 0] = s["scores"][b, w].double()
        v, i = rows.flatten().sort(descending=True, stable=True)
        k = min(case["K"], int((v[:case["K"]] > -math.inf).sum()))
        out["scores"][b, :k] = v[:k]
        out["parents"][b, :k] = (b * W + i[:k] // V).int()
        out["tokens"][b, :k] = (i[:k] % V).int()
    return out


def _exact_pages(case, s):
    tables, refs, lens = s["tables"].tolist(), s["refs"].tolist(), s["lens"].tolist()
    parents, page, S = s["parents"].tolist(), case["page"], len(tables)
    kids = {p: [c for c in range(S) if parents[c] == p] for p in range(S)}
    for p in range(S):
        if not kids[p]:
            for e in tables[p]:
                if e >= 0:
                    refs[e] -= 1
    spare, copies = iter([p for p, r in enumerate(refs) if r <= 0]), []
    new_tables, new_lens, granted = [], [], []
    for c in range(S):
        p = parents[c]
        if (p if p in kids[p] else kids[p][0]) == c:
            new_tables.append(list(tables[p]))
            new_lens.append(lens[p])
            granted.append(1)
            continue
        full, rest = divmod(lens[p], page)
        row = tables[p][:full] + [-1] * (len(tables[p]) - full)
        dst = next(spare, None) if rest else 0
        if dst is None:
            new_tables.append([-1] * len(row))
            new_lens.append(0)
            granted.append(0)
            continue
        if rest:
            copies.append((tables[p][full], dst))
            row[full] = dst
            refs[dst] = 1
        for e in tables[p][:full]:
            refs[e] += 1
        new_tables.append(row)
        new_lens.append(lens[p])
        granted.append(1)
    pages = _words(s["pages"])
    for t in pages:
        old = {src: t[:, src].clone() for src, _ in copies}
        for src, dst in copies:
            t[:, dst] = old[src]
    return dict(tables=_ints(new_tables), refs=_ints(refs), lengths=_ints(new_lens), granted=_ints(granted), pages=pages)


def _exact_cache(case, s):
    parents, lens, pages = s["parents"].tolist(), s["lens"].tolist(), []
    for t in _words(s["pages"]):
        new = t.clone()
        for c, p in enumerate(parents):
            new[c, :, :lens[p]] = t[p, :, :lens[p]]
        pages.append(new)
    return dict(lengths=_ints([lens[p] for p in parents]), pages=pages)


def _rows64(pool, pages, h, n):
    """The first n rows of head h over a list of pages, in 64 bits."""
    w, s, b = (t[pages, h].flatten(0, 1)[:n] for t in pool)
    w = w.long() & 0xFFFFFFFF
    nib = torch.stack([(w >> (4 * i)) & 15 for i in range(8)], -1).reshape(n, -1, 64).double()
    return torch.addcmul(b.double()[..., None], nib, s.double()[..., None]).reshape(n, -1)


def _exact_chunks(case, s):
    Hkv, G, W, sinks = case["Hkv"], case["Hq"] // case["Hkv"], case["window"], case["sinks"]
    pool, q = _words(s["pages"]), s["q_"].double()
    starts, lens, out = s["starts"].tolist(), s["lens"].tolist(), torch.zeros_like(s["q_"], dtype=torch.float64)
    for b, L in enumerate(lens):
        mine = slice(starts[b], starts[b + 1])
        n = mine.stop - mine.start
        pos, j = L - n + torch.arange(n, device="cuda")[:, None], torch.arange(L, device="cuda")[None]
        keep = (j <= pos) & ((pos - j < W) | (j < sinks) if W else True)
        for h in range(Hkv):
            k, v = (_rows64(pool[i:i + 3], s["tables"][b, :_pages(L, case["page"])].long(), h, L) for i in (0, 3))
            for i in range(h * G, h * G + G):
                out[mine, i] = torch.softmax((q[mine, i] @ k.t()).masked_fill(~keep, -math.inf), -1) @ v
    return out


def exact(case, seed):
    return {"select": _exact_select, "pages": _exact_pages, "cache": _exact_cache,
            "chunks": _exact_chunks}[case["kind"]](case, prepare(case, seed))
