"""The operators of a paged cache and the filtered draw in 64 bits, one sequence or row after the other (torch, on the tensors' device)."""
import numpy as np
import torch


def places(lens, starts):
    """(sequence, rows, positions) of every sequence with new tokens."""
    for b, n in enumerate(lens):
        rows = range(starts[b], starts[b + 1])
        if len(rows):
            yield b, rows, [n - len(rows) + i for i in range(len(rows))]


def attend(q, k, v, table, lens, starts, window, first, scale, want_sizes=False):
    """out [T, Hq, D] in 64 bits (rows of no sequence: NaN); with want_sizes also the sums of w |v| and, per row and head, the largest sum of
    |q_d k_d| scale, which rounding errors are measured by."""
    T, Hq, D = q.shape
    n_pages, Hkv, page, _ = k.shape
    out = torch.full((T, Hq, D), float("nan"), dtype=torch.float64, device=q.device)
    size, score_size = torch.zeros_like(out), torch.zeros(T, Hq, 1, dtype=torch.float64, device=q.device)
    table = table.cpu()
    for b, rows, pos in places(lens, starts):
        names = [int(x) if 0 <= int(x) < n_pages else -1 for x in table[b]]
        have = [j for j in range(min(lens[b], len(names) * page)) if names[j // page] >= 0]
        j = torch.tensor(have, dtype=torch.long, device=q.device)
        where = torch.tensor([names[x // page] for x in have], dtype=torch.long, device=q.device)
        for i, p in zip(rows, pos):
            seen = j <= p
            if window:
                seen &= (j > p - window) | (j < first)
            at = j[seen]
            if not len(at):
                out[i] = 0
                continue
            kk = k[where[seen], :, at % page].double()  # [n, Hkv, D]
            vv = v[where[seen], :, at % page].double()
            qq = q[i].double().view(Hkv, Hq // Hkv, D)
            s = torch.einsum("hgd,nhd->hgn", qq, kk) * scale
            w = torch.softmax(s, -1)
            w = torch.where((s == -torch.inf).all(-1, keepdim=True), torch.zeros_like(w), w)
            terms = w[..., None] * vv.transpose(0, 1)[:, None]
            out[i] = terms.sum(2).reshape(Hq, D)
            size[i] = (w[..., None] * vv.transpose(0, 1)[:, None].abs()).sum(2).reshape(Hq, D)
            score_size[i] = (torch.einsum("hgd,nhd->hgn", qq.abs(), kk.abs()) * scale).amax(-1).reshape(Hq, 1)
    return (out, size, score_size) if want_sizes else out


def append(qkv, table, lens, starts, Hq, Hkv, D, qgain, kgain, eps, theta, q, k, v):
    """q, k, v in 64 bits with the new rows in place (the others as given)."""
    q, k, v = q.double().clone(), k.double().clone(), v.double().clone()
    n_pages, page = k.shape[0], k.shape[2]
    rate = theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device=qkv.device) / D)
    table = table.cpu()
    for b, rows, pos in places(lens, starts):
        for i, p in zip(rows, pos):
            x = qkv[i].double().view(Hq + 2 * Hkv, D)
            h = x[:Hq + Hkv]
            if qgain is not None:
                h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
                h = h * torch.cat([qgain.double().expand(Hq, D), kgain.double().expand(Hkv, D)])
            c, s = torch.cos(p * rate), torch.sin(p * rate)
            a, e = h[:, :D // 2], h[:, D // 2:]
            h = torch.cat([a * c - e * s, e * c + a * s], -1)
            q[i] = h[:Hq]
            name = int(table[b, p // page]) if 0 <= p // page < table.shape[1] else -1
            if 0 <= name < n_pages:
                k[name, :, p % page], v[name, :, p % page] = h[Hq:], x[Hq + Hkv:]
    return q, k, v


def draw(x, u, temperature, top_k, top_p, min_p):
    """Token and share of one row of logits (numpy, 64 bits)."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    order = np.lexsort((np.arange(len(x)), -x))
    top = x[order[0]]
    if top == -np.inf:
        return -1, 0.0
    if not temperature > 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, 0.0) if top == np.inf else np.where(x == -np.inf, 0.0, np.exp((x - top) / temperature))
    keep = order[:top_k] if 0 < top_k < len(x) else order
    if top_p < 1:
        sums = np.cumsum(w[keep])
        keep = keep[:max(1, int(np.searchsorted(sums, top_p * sums[-1], side="left")) + 1)]
    if min_p > 0:
        keep = keep[w[keep] >= min(min_p, 1.0)]
    keep = np.sort(keep)
    sums = np.cumsum(w[keep])
    at = int(np.searchsorted(sums, min(max(u, 0.0), 1 - 2.0 ** -24) * sums[-1], side="right"))
    return int(keep[at]), float(w[keep[at]] / sums[-1])
