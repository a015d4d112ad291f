"""The operators of a paged cache, as cases that can be timed and compared.

One step of a serving program: the projections of the new tokens become normed, rotated queries and cache rows in pages (`append`), the new
tokens attend over the pages (`attend`), the logits become tokens (`sample`); when sequences fork, leave or are packed together, pages are
copied (`copy`).

A sequence's new tokens are rows of one packed array, its earlier keys and values lie in pages [page, kv head, slot, dim] that a table of page
numbers names. With `own` false every operator is computed from elementary torch operations, with `own` true by the framework.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"


# ------------------------------------------------------------------ what is measured
def listed():
    return [
        # two users of a small model, each one token further: latency
        dict(name="attend decode few", kind="attend", B=2, low=500, high=700, new=1, mix=False, Hq=16, Hkv=8, D=128, page=16, window=0, first=0),
        # a serving batch, contexts of 1k to 16k, one token each
        dict(name="attend decode batch", kind="attend", B=64, low=1024, high=16384, new=1, mix=False, Hq=32, Hkv=8, D=128, page=64, window=0, first=0),
        # long conversations under a sliding window whose first tokens stay visible, narrow heads
        dict(name="attend decode window", kind="attend", B=48, low=3000, high=32768, new=1, mix=False, Hq=32, Hkv=8, D=64, page=32, window=2048, first=4),
        # five drafted tokens per sequence are checked at once
        dict(name="attend drafts", kind="attend", B=16, low=1500, high=8192, new=5, mix=False, Hq=32, Hkv=8, D=128, page=16, window=0, first=0),
        # a chunk of a long document: few rows, many keys
        dict(name="attend chunk", kind="attend", B=1, low=16000, high=16000, new=512, mix=False, Hq=32, Hkv=8, D=128, page=16, window=0, first=0),
        # whole prompts of uneven length
        dict(name="attend prompts", kind="attend", B=4, low=683, high=2048, new=0, mix=False, Hq=32, Hkv=8, D=128, page=128, window=0, first=0),
        # the new tokens of a decode step enter the cache
        dict(name="append decode", kind="append", B=32, low=1000, high=2049, new=1, mix=False, Hq=32, Hkv=8, D=128, page=16, norm=True, theta=1e6),
        # prompts enter the cache, some of them in the middle of a page
        dict(name="append prompts", kind="append", B=8, low=1500, high=2901, new=1024, mix=False, Hq=32, Hkv=8, D=128, page=64, norm=True, theta=1e6),
        # a fork whose last pages are copied, keys and values of 28 layers
        dict(name="copy fork", kind="copy", pools=56, pages=64, page=16, Hkv=8, D=128, pairs=4),
        # a cache is packed together: pages move to the front
        dict(name="copy compaction", kind="copy", pools=72, pages=600, page=64, Hkv=8, D=128, pairs=151),
        # one user's next token
        dict(name="sample one", kind="sample", M=1, N=151936, dtype="fp32", temperature=0.7, top_k=20, top_p=0.95, min_p=0.0, mixed=False),
        # a batch whose users ask for different things, some of them greedy
        dict(name="sample batch", kind="sample", M=256, N=151936, dtype="fp32", temperature=0.9, top_k=50, top_p=0.9, min_p=0.05, mixed=True),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    kind = rng.choice(["attend"] * 6 + ["append", "copy", "sample", "sample"])
    heads = rng.choice([(32, 8), (16, 8), (12, 12), (8, 1), (32, 4), (14, 2)])
    D, page = rng.choice([128, 128, 64]), rng.choice([16, 32, 64, 128, 256])
    if kind == "attend":
        c = dict(kind=kind, D=D, page=page, Hq=heads[0], Hkv=heads[1], window=0, first=0, mix=False)
        if rng.random() < 0.35:
            c["window"], c["first"] = _log(rng, 20, 4096), rng.choice([0, 4, 150])
        how = rng.choice(["decode", "drafts", "chunk", "prompts", "mix"])
        high = _log(rng, 30, 2048 if how == "prompts" else 16384)
        low = max(1, high // rng.choice([1, 2, 8]))
        if how == "decode":
            B, new = _log(rng, 1, 64), 1
        elif how == "drafts":
            B, new = _log(rng, 1, 24), rng.randint(2, 9)
        elif how == "chunk":
            B, new = 1 if high > 4000 else rng.randint(1, 3), _log(rng, 17, 700)
        elif how == "prompts":
            B, new = rng.randint(1, 4), 0
        else:
            B, new = rng.randint(2, 9), _log(rng, 17, 300)
            c["mix"] = True
            high = min(high, 4096)
            low = min(low, high)
        return dict(c, B=B, low=low, high=high, new=new)
    if kind == "append":
        high = _log(rng, 40, 8192)
        new = rng.choice([1, 1, _log(rng, 2, 1200)])
        B = _log(rng, 1, 64) if new == 1 else _log(rng, 1, max(1, min(16, 8192 // new)))
        return dict(kind=kind, B=B, low=max(1, high // rng.choice([1, 4])), high=high, new=new, mix=B > 1 and rng.random() < 0.3, Hq=heads[0], Hkv=heads[1], D=D,
                    page=page, norm=rng.random() < 0.7, theta=rng.choice([1e4, 1e6]))
    if kind == "copy":
        pages = _log(rng, 8, 400)
        return dict(kind=kind, pools=rng.choice([1, 2, 24, 56, 72]), pages=pages, page=rng.choice([16, 64]), Hkv=heads[1], D=D, pairs=_log(rng, 1, max(1, pages // 2)))
    on = [rng.random() < 0.6 for _ in range(3)]
    return dict(kind=kind, M=_log(rng, 1, 200), N=_log(rng, 1000, 151936), dtype=rng.choice(["fp32", "fp32", "bf16"]), temperature=rng.choice([0.5, 0.8, 1.0, 1.3]),
                top_k=_log(rng, 2, 2000) if on[0] else 0, top_p=rng.choice([0.5, 0.8, 0.95, 0.99]) if on[1] else 1.0,
                min_p=rng.choice([0.02, 0.1]) if on[2] else 0.0, mixed=rng.random() < 0.3)


def _gen(seed, what):
    return torch.Generator(DEV).manual_seed((seed * 1000003 + what) & 0x7FFFFFFFFFFF)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)


def _lengths(case):
    """Length of every sequence, new tokens included, and the number of those; the same for every seed."""
    B, low, high = case["B"], case["low"], case["high"]
    lens = [high - (high - low) * i // max(1, B - 1) for i in range(B)]
    new = [min(n, case["new"] or n) for n in lens]
    if case["mix"]:
        new = new[:1] + [1] * (B - 1)
    return lens, new


def prepare(case, seed):
    s = dict(case)
    g = _gen(seed, 1)
    if case["kind"] == "sample":
        M, n = case["M"], case["N"]
        s["logits"] = torch.randn(M, n, generator=g, device=DEV) * 3
        if case["dtype"] == "bf16":
            s["logits"] = s["logits"].to(torch.bfloat16)
        s["u"] = torch.rand(M, generator=g, device=DEV)
        for k, t, off in (("temperature", torch.float32, 0.0), ("top_k", torch.int32, 0), ("top_p", torch.float32, 1.0), ("min_p", torch.float32, 0.0)):
            v = torch.full((M,), case[k], dtype=t, device=DEV)
            if case["mixed"]:  # each row goes without some of them; without a temperature it is greedy
                v = torch.where(torch.rand(M, generator=g, device=DEV) < (0.1 if k == "temperature" else 0.5), torch.full_like(v, off), v)
            s[k] = v
        s["out"], s["prob"] = torch.zeros(M, dtype=torch.int32, device=DEV), torch.zeros(M, device=DEV)
        return s
    if case["kind"] == "copy":
        s["cache"] = _randn(g, case["pools"], case["pages"], case["Hkv"], case["page"], case["D"])
        rng = np.random.default_rng([seed, 4])
        order = rng.permutation(case["pages"])[:2 * case["pairs"]].astype(np.int32)
        s["src"], s["dst"] = order[:case["pairs"]].copy(), order[case["pairs"]:].copy()
        s["addresses"] = np.array([s["cache"][i].data_ptr() for i in range(case["pools"])], np.uint64)
        return s
    lens, new = _lengths(case)
    per = [-(-n // case["page"]) for n in lens]
    ld = max(per)
    s["n_pages"] = sum(per) + 3
    places = torch.randperm(s["n_pages"], generator=g, device=DEV, dtype=torch.int32)
    table = torch.full((case["B"], ld), -1, dtype=torch.int32)
    held, at = places.cpu(), 0
    for b, n in enumerate(per):
        table[b, :n] = held[at:at + n]
        at += n
    s["table"], s["table_ld"] = table.to(DEV), ld
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["starts"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=DEV)
    s["T"], s["max_new"], s["max_len"] = sum(new), max(new), max(lens)
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    s["k"], s["v"] = (_randn(g, s["n_pages"], Hkv, case["page"], D) for _ in range(2))
    s["q"] = torch.zeros(s["T"], Hq, D, dtype=torch.bfloat16, device=DEV)
    if case["kind"] == "attend":
        s["q"] = _randn(g, s["T"], Hq, D)
        s["out"] = torch.zeros_like(s["q"])
    else:
        s["qkv"] = _randn(g, s["T"], (Hq + 2 * Hkv) * D)
        s["qgain"] = s["kgain"] = None
        if case["norm"]:
            s["qgain"], s["kgain"] = (1 + 0.1 * torch.randn(D, generator=g, device=DEV) for _ in range(2))
    return s


def run(s):
    if own:
        return _own(s)
    return {"attend": _attend, "append": _append, "copy": _copy, "sample": _sample}[s["kind"]](s)


# ------------------------------------------------------------------ the framework's calls
_kept = {}


def _own(s):
    from strict_b200 import native as N
    from strict_b200.kernel import Context
    if "ctx" not in _kept:
        _kept["ctx"] = Context(0)  # the program's one context
    L, h = N.lib(), _kept["ctx"].h
    p = lambda k: None if s[k] is None else s[k].data_ptr()  # noqa: E731
    if s["kind"] == "attend":
        N.check(L.strictb200_attn_paged(h, p("q"), p("k"), p("v"), p("table"), p("lens"), p("starts"), s["B"], s["T"], s["max_new"], s["max_len"], s["Hq"], s["Hkv"],
                                        s["D"], s["n_pages"], s["page"], s["table_ld"], s["window"], s["first"], s["D"] ** -0.5, p("out")))
        return s["out"]
    if s["kind"] == "append":
        N.check(L.strictb200_rope_qknorm_paged(h, p("qkv"), p("table"), p("lens"), p("starts"), s["B"], s["T"], s["Hq"], s["Hkv"], s["D"], p("qgain"), p("kgain"), 1e-6,
                                               s["theta"], s["n_pages"], s["page"], s["table_ld"], p("q"), p("k"), p("v")))
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    if s["kind"] == "copy":
        N.check(L.strictb200_pages_copy(h, N.ptr(s["addresses"]), s["pools"], s["pages"], s["page"] * s["Hkv"] * s["D"] * 2, N.ptr(s["src"]), N.ptr(s["dst"]), s["pairs"]))
        return s["cache"]
    N.check(L.strictb200_sample(h, p("logits"), 1 if s["dtype"] == "fp32" else 0, s["M"], s["N"], s["N"], p("u"), p("temperature"), p("top_k"), p("top_p"), p("min_p"),
                                p("out"), p("prob")))
    return {"token": s["out"], "prob": s["prob"]}


# ------------------------------------------------------------------ plain forms
def _places(s):
    """Sequence and position of every new row."""
    rows = torch.arange(s["T"], device=DEV)
    seq = torch.searchsorted(s["starts"][1:].long(), rows, right=True)
    return seq, s["lens"].long()[seq] - s["starts"].long()[seq + 1] + rows


def _attend(s):
    """softmax(q k^T scale) v over the keys j <= position with j > position - window or j < first."""
    B, Hq, Hkv, D, S = s["B"], s["Hq"], s["Hkv"], s["D"], s["max_new"]
    keys, values = (s[x][s["table"].long().clamp(min=0)].float().transpose(1, 2).reshape(B, Hkv, -1, D) for x in ("k", "v"))
    seq, pos = _places(s)
    row = torch.arange(s["T"], device=DEV) - s["starts"].long()[seq]
    q = torch.zeros(B, S, Hq, D, device=DEV)
    q[seq, row] = s["q"].float()
    q = q.view(B, S, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    score = (q @ keys.transpose(-1, -2)).view(B, Hkv, Hq // Hkv, S, -1) * s["D"] ** -0.5
    at = torch.full((B, S), -1, device=DEV)
    at[seq, row] = pos
    j = torch.arange(keys.shape[2], device=DEV)
    seen = j <= at[..., None]
    if s["window"]:
        seen &= (j > at[..., None] - s["window"]) | (j < s["first"])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top == -math.inf, 0, top))
    o = (w.view(B, Hkv, -1, keys.shape[2]) @ values).view(B, Hkv, Hq // Hkv, S, D) / w.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(B, S, Hq, D)[seq, row].to(torch.bfloat16)


def _append(s):
    """RMS norm per head, rotation of the pairs (i, i + D / 2) by position * theta^(-2 i / D), rows into pages."""
    Hq, Hkv, D = s["Hq"], s["Hkv"], s["D"]
    x = s["qkv"].float().view(s["T"], Hq + 2 * Hkv, D)
    seq, pos = _places(s)
    turn = pos[:, None].double() * s["theta"] ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    cos, sin = torch.cos(turn).float()[:, None], torch.sin(turn).float()[:, None]

    def turned(h, gain):
        if gain is not None:
            h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * gain
        a, b = h[..., :D // 2], h[..., D // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(torch.bfloat16)

    page, slot = s["table"][seq, pos // s["page"]].long(), pos % s["page"]
    s["q"].copy_(turned(x[:, :Hq], s["qgain"]))
    s["k"][page, :, slot] = turned(x[:, Hq:Hq + Hkv], s["kgain"])
    s["v"][page, :, slot] = x[:, Hq + Hkv:].to(torch.bfloat16)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _copy(s):
    s["cache"][:, torch.from_numpy(s["dst"]).to(DEV).long()] = s["cache"][:, torch.from_numpy(s["src"]).to(DEV).long()]
    return s["cache"]


def _sample(s):
    """Tokens by falling logit, the lower index first: the first top_k, of those the shortest beginning that holds top_p of their mass, of those
    with min_p of the largest probability; drawn in the order of the indices by u."""
    x = s["logits"].double()
    greedy = s["temperature"] <= 0
    heat = torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    w = torch.exp((x - x.amax(-1, keepdim=True)) / heat)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    place = torch.arange(s["N"], device=DEV)
    sorted_w = w.gather(-1, order)
    keep = (place < s["top_k"][:, None]) | (s["top_k"][:, None] <= 0)
    sorted_w = torch.where(keep, sorted_w, 0.0)
    sums = sorted_w.cumsum(-1)
    keep &= (sums - sorted_w < s["top_p"].double()[:, None] * sums[:, -1:]) | (s["top_p"][:, None] >= 1)
    keep &= sorted_w >= s["min_p"].double()[:, None]
    keep &= (place == 0) | ~greedy[:, None]
    w = torch.where(torch.zeros_like(keep).scatter(-1, order, keep), w, 0.0)
    sums = w.cumsum(-1)
    token = torch.searchsorted(sums, s["u"].double()[:, None] * sums[:, -1:], right=True)
    return {"token": token[:, 0].to(torch.int32), "prob": (w.gather(-1, token) / sums[:, -1:])[:, 0].float()}


# ------------------------------------------------------------------ the same in 64 bits, one sequence or row after the other
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        moved = s["cache"].clone()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            moved[:, b] = s["cache"][:, a]
        return moved
    if case["kind"] == "sample":
        tokens = []
        for m in range(case["M"]):
            x = s["logits"][m].cpu().double().numpy()
            heat, k, p, least = (s[n][m].double().item() for n in ("temperature", "top_k", "top_p", "min_p"))
            if heat <= 0:
                tokens.append(1.0)
                continue
            e = np.exp((x - x.max()) / heat)
            by = np.lexsort((np.arange(len(x)), -x))
            if 0 < k < len(x):
                by = by[:int(k)]
            if p < 1:
                c = np.cumsum(e[by])
                by = by[:int(np.searchsorted(c, p * c[-1], side="left")) + 1]
            by = np.sort(by[e[by] >= least])
            c = np.cumsum(e[by])
            at = int(np.searchsorted(c, s["u"][m].double().item() * c[-1], side="right"))
            tokens.append(e[by[at]] / c[-1])
        return {"token": None, "prob": torch.tensor(tokens, dtype=torch.float64)}
    lens, new = _lengths(case)
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    out, first = torch.empty(s["T"], Hq, D, dtype=torch.float64, device=DEV), 0
    if case["kind"] == "append":
        kp, vp = s["k"].double(), s["v"].double()
    for b in range(case["B"]):
        L, n = lens[b], new[b]
        rows, first = slice(first, first + n), first + n
        pos = torch.arange(L - n, L, device=DEV)
        names = s["table"][b, :-(-L // page)].long()
        if case["kind"] == "append":
            x = s["qkv"][rows].double().view(n, -1, D)
            z = torch.complex(x[:, :Hq + Hkv, :D // 2], x[:, :Hq + Hkv, D // 2:])
            if case["norm"]:
                gain = torch.cat([s["qgain"].double().expand(Hq, D), s["kgain"].double().expand(Hkv, D)])
                size = torch.sqrt((z.real ** 2 + z.imag ** 2).sum(-1, keepdim=True) / D + 1e-6)
                z = torch.complex(z.real * gain[:, :D // 2], z.imag * gain[:, D // 2:]) / size
            rate = torch.exp(-math.log(case["theta"]) * torch.arange(D // 2, device=DEV, dtype=torch.float64) * 2 / D)
            z = z * torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos.double()[:, None] * rate)[:, None]
            y = torch.cat([z.real, z.imag], -1)
            out[rows] = y[:, :Hq]
            kp[names[pos // page], :, pos % page] = y[:, Hq:]
            vp[names[pos // page], :, pos % page] = x[:, Hq + Hkv:]
            continue
        for h in range(Hkv):
            kk, vv = (s[t][names, h].reshape(-1, D)[:L].double() for t in ("k", "v"))
            j = torch.arange(L, device=DEV)
            hidden = j[None] > pos[:, None]
            if case["window"]:
                hidden |= (j[None] <= pos[:, None] - case["window"]) & (j[None] >= case["first"])
            for i in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                a = s["q"][rows, i].double() @ kk.T / math.sqrt(D)
                a[hidden] = -math.inf
                out[rows, i] = torch.softmax(a, -1) @ vv
    return out if case["kind"] == "attend" else {"q": out, "k": kp, "v": vp}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "sample":
        size = case["M"] * case["N"]
        return {"bytes": size * (4 if case["dtype"] == "fp32" else 2) + 28 * case["M"], "flops": 2 * size}
    if case["kind"] == "copy":
        return {"bytes": 2 * case["pools"] * case["pairs"] * case["page"] * case["Hkv"] * case["D"] * 2 + 8 * (case["pools"] + case["pairs"]), "flops": 0}
    lens, new = _lengths(case)
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "append":
        return {"bytes": 4 * sum(new) * (Hq + 2 * Hkv) * D, "flops": 10 * sum(new) * (Hq + Hkv) * D}
    W, F = case["window"], case["first"]
    keys = pairs = 0
    for L, n in zip(lens, new):
        low = max(0, L - n - W + 1) if W else 0  # first key in the window of the first new token
        keys += L - low + min(F, low)
        for p in range(L - n, L):
            at = max(0, p - W + 1) if W else 0
            pairs += p + 1 - at + min(F, at)
    return {"bytes": 4 * sum(new) * Hq * D + 4 * keys * Hkv * D, "flops": 4 * pairs * Hq * D}
