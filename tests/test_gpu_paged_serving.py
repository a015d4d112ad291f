"""The operators of a paged cache as a serving loop uses them: prompts, decode steps, forks, drafts that are cut back, sequences that leave, packing. Every
step's rows are checked against 64-bit forms over a record of what each sequence has appended, so pages that were shared, copied or moved have to hold
what they held. And the sizes at which the attention changes its kernel."""
import numpy as np
import pytest
import torch

import paged_plain as plain
from strict_b200 import native as N
from strict_b200.kernel import Context
from test_gpu_paged import Cache, HALF, L, ptr

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


class Serving:
    """Layers of one paged cache, sequences as lists of pages with counts of who holds them, and a record of every row that was appended."""

    def __init__(self, ctx, layers, Hq, Hkv, D, page, n_pages, window, first, seed):
        self.ctx, self.layers, self.Hq, self.Hkv, self.D, self.page, self.n_pages, self.window, self.first = ctx, layers, Hq, Hkv, D, page, n_pages, window, first
        self.g = torch.Generator("cuda").manual_seed(seed)
        self.pool = torch.full((2 * layers, n_pages, Hkv, page, D), float("nan"), dtype=BF16, device="cuda")
        self.held = np.zeros(n_pages, int)
        self.pages, self.length, self.record = {}, {}, {}
        vocab = 700
        rand = lambda *s: torch.randn(*s, generator=self.g, device="cuda")  # noqa: E731
        self.embed = rand(vocab, 64)
        self.wqkv = [rand(64, (Hq + 2 * Hkv) * D) for _ in range(layers)]
        self.wo = [rand(Hq * D, 64) / (Hq * D) ** 0.5 for _ in range(layers)]
        self.gains = [1 + 0.2 * rand(D) for _ in range(2)]
        self.vocab, self.rng = vocab, np.random.default_rng(seed)

    def take(self):
        p = int(np.flatnonzero(self.held == 0)[-1])  # from the end, so that packing has something to do
        self.held[p] = 1
        return p

    def copy(self, src, dst):
        where = np.array([self.pool[i].data_ptr() for i in range(2 * self.layers)], np.uint64)
        N.check(L().strictb200_pages_copy(self.ctx.h, N.ptr(where), 2 * self.layers, self.n_pages, self.Hkv * self.page * self.D * 2, N.ptr(np.array(src, np.int32)),
                                          N.ptr(np.array(dst, np.int32)), len(src)))

    def open(self, s):
        self.pages[s], self.length[s], self.record[s] = [], 0, [[[], []] for _ in range(self.layers)]

    def fork(self, s, to):
        """Full pages are shared; the last one, which both will write into, is copied."""
        self.pages[to], self.length[to] = list(self.pages[s]), self.length[s]
        self.record[to] = [[list(x) for x in layer] for layer in self.record[s]]
        for p in self.pages[to]:
            self.held[p] += 1
        if self.length[s] % self.page:
            old, new = self.pages[to][-1], self.take()
            self.held[old] -= 1
            self.pages[to][-1] = new
            self.copy([old], [new])

    def close(self, s):
        for p in self.pages.pop(s):
            self.held[p] -= 1
        del self.length[s], self.record[s]

    def trim(self, s, n):
        self.length[s] = n
        while len(self.pages[s]) > -(-n // self.page):
            self.held[self.pages[s].pop()] -= 1
        for layer in self.record[s]:
            for x in layer:
                del x[n:]

    def pack(self):
        """Used pages move to the front."""
        used = int((self.held > 0).sum())
        src = [p for p in range(used, self.n_pages) if self.held[p]]
        dst = [p for p in range(used) if not self.held[p]]
        self.copy(src, dst)
        name = {a: b for a, b in zip(src, dst)}
        for s in self.pages:
            self.pages[s] = [name.get(p, p) for p in self.pages[s]]
        for a, b in name.items():
            self.held[b], self.held[a] = self.held[a], 0
        torch.cuda.synchronize()
        self.ctx.synchronize()
        self.pool[:, used:] = float("nan")
        return len(src)

    def step(self, new):
        """new: tokens per sequence. Returns the next token of each, drawn from the logits of its last row."""
        names = list(new)
        for s in names:
            self.length[s] += len(new[s])
            while len(self.pages[s]) * self.page < self.length[s]:
                self.pages[s].append(self.take())
        ld = max(len(self.pages[s]) for s in names) + 1
        table = torch.full((len(names), ld), -1, dtype=torch.int32)
        for i, s in enumerate(names):
            table[i, :len(self.pages[s])] = torch.tensor(self.pages[s], dtype=torch.int32)
        lens = [self.length[s] for s in names]
        starts = np.concatenate([[0], np.cumsum([len(new[s]) for s in names])]).tolist()
        T = starts[-1]
        table, d_lens, d_starts = table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor(starts, dtype=torch.int32, device="cuda")
        x = self.embed[torch.tensor(sum((list(new[s]) for s in names), []), device="cuda")]
        sizes = (self.n_pages, self.page, ld)
        for l in range(self.layers):
            k, v = self.pool[2 * l], self.pool[2 * l + 1]
            qkv = (x @ self.wqkv[l]).to(BF16)
            q, out = torch.zeros(T, self.Hq, self.D, dtype=BF16, device="cuda"), torch.zeros(T, self.Hq, self.D, dtype=BF16, device="cuda")
            torch.cuda.synchronize()
            # on the context's stream one after the other, nothing in between waits
            N.check(L().strictb200_rope_qknorm_paged(self.ctx.h, ptr(qkv), ptr(table), ptr(d_lens), ptr(d_starts), len(names), T, self.Hq, self.Hkv, self.D, ptr(self.gains[0]),
                                                     ptr(self.gains[1]), 1e-6, 1e4, *sizes, ptr(q), ptr(k), ptr(v)))
            N.check(L().strictb200_attn_paged(self.ctx.h, ptr(q), ptr(k), ptr(v), ptr(table), ptr(d_lens), ptr(d_starts), len(names), T, max(len(new[s]) for s in names),
                                              max(lens), self.Hq, self.Hkv, self.D, *sizes, self.window, self.first, self.D ** -0.5, ptr(out)))
            self.ctx.synchronize()
            self.ctx.device_status()
            self.check(l, names, lens, starts, qkv, q, out)
            x = x + out.float().reshape(T, -1) @ self.wo[l]
        last = torch.tensor(starts[1:], device="cuda") - 1
        logits = (x[last] @ self.embed.T).contiguous()
        u, temperature = self.rng.random(len(names), np.float32), np.array([0.0 if i % 3 == 2 else 2.0 for i in range(len(names))], np.float32)
        k, p = np.full(len(names), 40, np.int32), np.full(len(names), 0.95, np.float32)
        dev = [torch.from_numpy(a).cuda() for a in (u, temperature, k, p)]
        tokens = torch.zeros(len(names), dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        N.check(L().strictb200_sample(self.ctx.h, ptr(logits), 1, len(names), self.vocab, self.vocab, *[ptr(a) for a in dev], None, ptr(tokens), None))
        self.ctx.synchronize()
        host = logits.cpu().numpy()
        want = [plain.draw(host[i], float(u[i]), float(temperature[i]), 40, float(p[i]), 0.0)[0] for i in range(len(names))]
        assert tokens.tolist() == want
        return dict(zip(names, want))

    def check(self, l, names, lens, starts, qkv, q, out):
        D = self.D
        for i, s in enumerate(names):
            n, rows = lens[i], slice(starts[i], starts[i + 1])
            m = starts[i + 1] - starts[i]
            # the appended rows against the projection, on a cache of one sequence that lies in order
            flat = torch.zeros(1, self.Hkv, n, D, dtype=BF16, device="cuda")
            one = torch.zeros(1, 1, dtype=torch.int32)
            wq, wk, wv = plain.append(qkv[rows], one, [n], [0, m], self.Hq, self.Hkv, D, *self.gains, 1e-6, 1e4, q[rows], flat, flat)
            got = [torch.cat([self.pool[2 * l + x, p] for p in self.pages[s]], 1)[:, :n].transpose(0, 1) for x in (0, 1)]  # [n, Hkv, D]
            for a, w, pair in ((q[rows], wq, True), (got[0][n - m:], wk[0, :, n - m:].transpose(0, 1), True), (got[1][n - m:], wv[0, :, n - m:].transpose(0, 1), False)):
                other = torch.cat([w[..., D // 2:], w[..., :D // 2]], -1).abs() if pair else 0
                bound = HALF * w.abs() + (w.abs() + other) * ((D + 8) * 2.0 ** -24 + 2 * np.pi * 2.0 ** -24)
                assert ((a.double() - w).abs() <= bound).all()
            # earlier rows are what this sequence appended, wherever its pages have been since
            for x in (0, 1):
                rec = self.record[s][l][x]
                assert len(rec) == n - m and all(torch.equal(got[x][j], r) for j, r in enumerate(rec))
                rec.extend(got[x][j].clone() for j in range(n - m, n))
            keys, values = (g.transpose(0, 1)[None].contiguous() for g in got)
            want, size, scores = plain.attend(q[rows], keys, values, one, [n], [0, m], self.window, self.first, D ** -0.5, True)
            bound = HALF * want.abs() + size * (2.0 ** -15 + 2 * scores * (D + 2) * 2.0 ** -24 + 2 * n * 2.0 ** -24) + 1e-30
            assert ((out[rows].double() - want).abs() <= bound * (1 + HALF)).all(), (l, s)


@pytest.mark.parametrize("Hq,Hkv,D,page,window,first", [(8, 2, 128, 16, 0, 0), (6, 6, 64, 32, 40, 4), (16, 1, 128, 64, 0, 0)])
def test_serving(ctx, Hq, Hkv, D, page, window, first):
    S = Serving(ctx, 2, Hq, Hkv, D, page, 40, window, first, seed=Hq)
    prompt = lambda n: S.rng.integers(0, S.vocab, n).tolist()  # noqa: E731
    for s in "abc":
        S.open(s)
    after = S.step({"a": prompt(75), "b": prompt(16), "c": prompt(1)})
    for _ in range(3):
        after = S.step({s: [t] for s, t in after.items()})
    S.fork("a", "d")
    S.fork("b", "e")
    S.open("f")
    # one call with everything: decode steps, both ends of the forks on tokens of their own, a prompt's first chunk
    after = S.step({"a": [after["a"]], "b": [after["b"]], "c": [after["c"]], "d": [1], "e": [2], "f": prompt(50)})
    after = S.step({**{s: [t] for s, t in after.items()}, "f": prompt(33)})
    S.close("b")
    S.close("c")
    assert S.pack() > 0
    # drafts of four, of which two are taken
    drafted = S.step({s: [t] + prompt(3) for s, t in after.items() if s in S.pages})
    for s in drafted:
        S.trim(s, S.length[s] - 2)
    S.open("g")
    after = S.step({**{s: [t] for s, t in drafted.items()}, "g": prompt(130)})
    for _ in range(2):
        after = S.step({s: [t] for s, t in after.items()})
    for s in list(S.pages):
        S.close(s)
    assert (S.held == 0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,new", [(4, 2), (3, 3), (8, 2), (4, 4), (17, 1), (4, 5), (32, 1), (11, 3), (1, 16), (1, 17), (16, 8), (1, 128), (1, 129), (128, 1), (127, 2), (2, 64), (2, 65)])
def test_where_kernels_change(ctx, D, G, new):
    """Rows per sequence and key/value head around 8, 16, 128 and 256, with few keys and with many."""
    lens = [new, new + 3, 130 + new, 700]
    Cache(lens, [new, new, new, max(1, new // 2)], 2, D, 16, seed=G).check(ctx, G)
    Cache([1300, new + 1], [min(new, 9), min(new, 9)], 2, D, 16, seed=G).check(ctx, G)


@pytest.mark.parametrize("B", [33, 150, 700])
@pytest.mark.parametrize("new", [1, 7, 40])
def test_many_uneven_sequences(ctx, B, new):
    rng = np.random.default_rng(B + new)
    lens = [int(x) for x in np.exp(rng.uniform(0, np.log(260), B))]
    news = [min(n, int(rng.integers(0, new + 1))) for n in lens]
    news[B // 2], lens[B // 2] = new, max(new, lens[B // 2])
    Cache(lens, news, 2, 64, 16, seed=B, front=1, behind=2).check(ctx, 8)


def test_many_sequences_with_many_keys(ctx):
    """More than 128 sequences of one tile, the keys of each in two shares."""
    lens = [1400 if b % 40 == 0 else 3 + b % 50 for b in range(170)]
    Cache(lens, [3 if b % 7 else 0 for b in range(170)], 1, 128, 64, seed=1).check(ctx, 8)


@pytest.mark.parametrize("new", [1, 3, 5])
def test_uneven_lengths_in_parts(ctx, new):
    """A long sequence sets how keys are cut; the short ones have parts without any."""
    c = Cache([6000, new, 100, 1025, 63 + new], [new] * 5, 1, 128, 32, seed=new)
    c.check(ctx, 4)


def test_two_contexts(ctx):
    """Calls of two contexts, each with its stream and its scratch, run at the same time."""
    other = Context(0)
    pairs = []
    for i, x in enumerate((ctx, other)):
        for new in (2, 9):
            c = Cache([1500, 700, 30], [new] * 3, 2, 128, 16, seed=10 * i + new)
            q = torch.randn(c.T, 8, 128, generator=c.g, device="cuda").to(BF16)
            pairs.append((x, c, q, c.attend(x, q), [torch.full_like(q, 7.0) for _ in range(10)], new))
            c.compare(q, pairs[-1][3])
    torch.cuda.synchronize()
    for r in range(10):
        for x, c, q, _, outs, new in pairs:
            N.check(L().strictb200_attn_paged(x.h, ptr(q), ptr(c.k), ptr(c.v), ptr(c.table), ptr(c.d_lens), ptr(c.d_starts), 3, c.T, new, 1500, 8, 2, 128, c.n_pages, 16,
                                              c.ld, 0, 0, 128 ** -0.5, ptr(outs[r])))
    ctx.synchronize()
    other.synchronize()
    for _, _, _, want, outs, _ in pairs:
        assert all(torch.equal(o, want) for o in outs)
    other.dispose()


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 1, 64), (10, 2, 128), (128, 1, 128)])
@pytest.mark.parametrize("T", [591, 593, 1300, 10001])
def test_appends_of_many_tokens(ctx, Hq, Hkv, D, T):
    """A block takes one to sixteen tokens: the places of rows in front of, between and behind sequences, and of empty sequences."""
    lens, new = [T // 2, 5, 0, T - T // 2 - 8 + 64], [T // 2 - 2, 0, 0, T - T // 2 - 8]
    c = Cache(lens, new, Hkv, D, 64, seed=T, rest=0.0, front=3, behind=T - 3 - sum(new))
    c.table[0, 1] = -1
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=c.g, device="cuda").to(BF16)
    q = torch.full((T, Hq, D), 7.0, dtype=BF16, device="cuda")
    k, v = c.k.clone(), c.v.clone()
    torch.cuda.synchronize()
    N.check(L().strictb200_rope_qknorm_paged(ctx.h, ptr(qkv), ptr(c.table), ptr(c.d_lens), ptr(c.d_starts), 4, T, Hq, Hkv, D, None, None, 0.0, 1e4, c.n_pages, 64, c.ld,
                                             ptr(q), ptr(c.k), ptr(c.v)))
    ctx.synchronize()
    inside = torch.zeros(T, dtype=torch.bool, device="cuda")
    inside[c.starts[0]:c.starts[-1]] = True
    assert (q[~inside] == 7.0).all()
    rows = torch.arange(T, device="cuda")
    seq = torch.searchsorted(c.d_starts[1:].long(), rows, right=True).clamp(max=3)
    pos = c.d_lens.long()[seq] - c.d_starts.long()[seq + 1] + rows
    x = qkv.double().view(T, Hq + 2 * Hkv, D)
    rate = 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    cs, sn = torch.cos(pos[:, None] * rate)[:, None], torch.sin(pos[:, None] * rate)[:, None]
    a, e = x[:, :Hq + Hkv, :D // 2], x[:, :Hq + Hkv, D // 2:]
    w = torch.cat([a * cs - e * sn, e * cs + a * sn], -1)
    bound = HALF * w.abs() + (w.abs() + torch.cat([w[..., D // 2:], w[..., :D // 2]], -1).abs()) * (8 + 2 * np.pi) * 2.0 ** -24
    assert ((q.double() - w[:, :Hq]).abs() <= bound[:, :Hq])[inside].all()
    name = c.table.long()[seq, (pos // 64).clamp(0, c.ld - 1)]
    wrote = inside & (pos // 64 < c.ld) & (name >= 0)
    kk, vv = c.k[name[wrote], :, pos[wrote] % 64], c.v[name[wrote], :, pos[wrote] % 64]
    assert ((kk.double() - w[wrote][:, Hq:]).abs() <= bound[wrote][:, Hq:]).all() and torch.equal(vv, qkv.view(T, -1, D)[wrote][:, Hq + Hkv:])
    k[name[wrote], :, pos[wrote] % 64], v[name[wrote], :, pos[wrote] % 64] = kk, vv
    assert torch.equal(k, c.k) and torch.equal(v, c.v), "nothing else is written"


def test_many_drafts(ctx):
    """So many rows that two shares of each would take more scratch than they may."""
    B, G = 1100, 16
    rng = np.random.default_rng(3)
    lens = [int(x) for x in rng.integers(2, 60, B)]
    c = Cache(lens, [2] * B, 8, 128, 16, seed=3)
    q = torch.randn(c.T, 8 * G, 128, generator=c.g, device="cuda").to(BF16)
    out = c.attend(ctx, q)
    few = list(range(0, B, 97)) + [B - 1]
    for b in few:
        rows = slice(c.starts[b], c.starts[b + 1])
        want, size, scores = plain.attend(q[rows], c.k, c.v, c.table[b:b + 1], lens[b:b + 1], [0, 2], 0, 0, 128 ** -0.5, True)
        bound = HALF * want.abs() + size * (2.0 ** -15 + 2 * scores * 130 * 2.0 ** -24 + 2 * 60 * 2.0 ** -24) + 1e-30
        assert ((out[rows].double() - want).abs() <= bound * (1 + HALF)).all(), b
