"""The operators of a paged cache against their plain forms in 64 bits (paged_plain.py)."""
import ctypes

import numpy as np
import pytest
import torch

import paged_plain as plain
from strict_b200 import native as N

pytestmark = pytest.mark.gpu
BF16, HALF = torch.bfloat16, torch.finfo(torch.bfloat16).eps / 2  # half a step, relative


def L():
    return N.lib()


def ptr(t):
    return None if t is None else t.data_ptr()


class Cache:
    """Pages of B sequences in random places, `ld` table columns; pages no sequence holds, and slots behind a length, are filled with `rest`."""

    def __init__(self, lens, new, Hkv, D, page, seed=0, rest=float("nan"), extra=2, ld=None, front=0, behind=0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.lens, self.g = list(lens), g
        self.starts = [front]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.T = self.starts[-1] + behind
        per = [-(-n // page) for n in lens]
        self.ld = ld or max(1, max(per, default=1))
        self.n_pages, self.page = sum(per) + extra, page
        order = torch.randperm(self.n_pages, generator=g, device="cuda").tolist()
        self.k, self.v = (torch.randn(self.n_pages, Hkv, page, D, generator=g, device="cuda").to(BF16) for _ in range(2))
        table = torch.full((max(1, len(self.lens)), self.ld), -1, dtype=torch.int32)
        held, at = torch.zeros(self.n_pages, page, dtype=torch.bool), 0
        for b, n in enumerate(per):
            for i in range(min(n, self.ld)):
                table[b, i] = order[at + i]
                held[order[at + i], :min(page, lens[b] - i * page)] = True
            at += n
        hidden = ~held.cuda()[:, None, :, None].expand_as(self.k)
        self.k[hidden], self.v[hidden] = rest, rest
        self.table = table.cuda()
        self.d_lens = torch.tensor(self.lens or [0], dtype=torch.int32, device="cuda")
        self.d_starts = torch.tensor(self.starts, dtype=torch.int32, device="cuda")

    def attend(self, ctx, q, window=0, first=0, scale=None, out=None, max_new=None, max_len=None):
        Hkv, D = self.k.shape[1], self.k.shape[3]
        out = torch.full_like(q, 7.0) if out is None else out
        new = [b - a for a, b in zip(self.starts, self.starts[1:])]
        torch.cuda.synchronize()
        N.check(L().strictb200_attn_paged(ctx.h, ptr(q), ptr(self.k), ptr(self.v), ptr(self.table), ptr(self.d_lens), ptr(self.d_starts), len(self.lens), self.T,
                                          max(new, default=0) if max_new is None else max_new, max(self.lens, default=0) if max_len is None else max_len,
                                          q.shape[1], Hkv, D, self.n_pages, self.page, self.ld, window, first, D ** -0.5 if scale is None else scale, ptr(out)))
        ctx.synchronize()
        ctx.device_status()
        return out

    def check(self, ctx, G, window=0, first=0, scale=None, amp=1.0, **kw):
        Hkv, D = self.k.shape[1], self.k.shape[3]
        q = (torch.randn(self.T, Hkv * G, D, generator=self.g, device="cuda") * amp).to(BF16)
        out = self.attend(ctx, q, window, first, scale, **kw)
        self.compare(q, out, window, first, scale)
        return q, out

    def compare(self, q, out, window=0, first=0, scale=None):
        D = q.shape[2]
        want, size, scores = plain.attend(q, self.k, self.v, self.table, self.lens, self.starts, window, first, D ** -0.5 if scale is None else scale, True)
        none = want.isnan().all(-1)  # rows of no sequence
        rows = torch.zeros(self.T, dtype=torch.bool, device="cuda")
        rows[self.starts[0]:self.starts[-1]] = True
        assert (out[~rows] == 7.0).all(), "rows of no sequence are left as they are"
        # The output's rounding; the softmax weights enter the product in two bf16 terms (2^-16); a score's products are exact in fp32, its D sums and the
        # scaling are off by (D + 2) 2^-24 of the sum of magnitudes, and so are, twice (weight and sum), the logarithms of the weights; running sums over the
        # keys, at most 2^-24 for each of them and their rescalings.
        n = max(self.lens, default=1)
        bound = HALF * want.abs() + size * (2.0 ** -15 + 2 * scores * (D + 2) * 2.0 ** -24 + 2 * n * 2.0 ** -24) + 1e-30
        err = (out.double() - want).abs()
        bad = (err > bound * (1 + HALF)) & rows[:, None, None] & ~none[..., None]
        assert not bad.any(), f"{int(bad.sum())} values, worst {float((err / bound)[rows].nan_to_num(0).max()):.2f} of the bound at {bad.nonzero()[0].tolist()}"
        assert torch.equal(out[rows].isnan(), want[rows].isnan())


HEADS = [(8, 4, 128), (2, 1, 64), (3, 2, 128), (1, 7, 64), (1, 16, 128)]


@pytest.mark.parametrize("Hkv,G,D", HEADS)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_decode_steps(ctx, Hkv, G, D, page):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 777]
    Cache(lens, [1] * len(lens), Hkv, D, page, seed=page + G).check(ctx, G)


@pytest.mark.parametrize("Hkv,G,D", HEADS + [(1, 40, 128), (1, 128, 64), (2, 5, 128)])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_chunks(ctx, Hkv, G, D, page):
    """Few and many new tokens, whole prompts, sequences without new tokens, sequences without any."""
    lens, new = [5, 130, 0, 260, 129, 40, 300], [5, 3, 0, 140, 1, 0, 33]
    Cache(lens, new, Hkv, D, page, seed=page + G).check(ctx, G)


@pytest.mark.parametrize("new", [1, 2, 7, 40])
@pytest.mark.parametrize("window,first", [(1, 0), (5, 2), (64, 0), (100, 4), (128, 130), (200, 64), (1000, 1)])
@pytest.mark.parametrize("page", [16, 64])
def test_windows(ctx, new, window, first, page):
    lens = [1, 60, 129, 333, 700, 411]
    Cache(lens, [min(n, new) for n in lens], 2, 128, page, seed=window).check(ctx, 4, window, first)


def test_window_leaves_freed_pages_alone(ctx):
    """Pages that no row sees may be gone: their entries name nothing, or a page of somebody else that holds NaN."""
    for new in (1, 3, 150):
        c = Cache([900, 700], [new, new], 2, 128, 16, seed=new)
        q, out = c.check(ctx, 4, 200, 20)
        for b, n in enumerate(c.lens):
            first_seen = n - new - 200 + 1
            for i in range(2, max(2, first_seen // 16)):  # positions 32 .. first_seen - 1 at most
                c.table[b, i] = -1 if i % 2 else c.n_pages + 5
        assert torch.equal(c.attend(ctx, q, 200, 20), out)
        c.compare(q, out, 200, 20)


def test_entries_that_name_no_page_hide_their_keys(ctx):
    for new in (1, 4, 130):
        c = Cache([300, 513, 140], [new] * 3, 2, 128, 16, seed=new)
        c.table[0, 0], c.table[0, 7], c.table[1, :] = -1, c.n_pages, -7  # sequence 1 sees nothing: zeros
        c.table[2, 3] = -2 ** 31
        q, out = c.check(ctx, 4)
        assert (out[c.starts[1]:c.starts[2]] == 0).all()


def test_lengths_beyond_the_table(ctx):
    for new in (1, 150):
        Cache([700, 200], [new, new], 2, 128, 16, seed=new, ld=20).check(ctx, 2)  # 320 positions are there


def test_rows_in_front_of_their_sequence(ctx):
    """More new rows than tokens: the rows at negative positions see nothing."""
    c = Cache([3, 40], [5, 9], 2, 64, 16, seed=1)
    q, out = c.check(ctx, 4)
    assert (out[:2] == 0).all()


def test_rows_of_no_sequence_stay(ctx):
    Cache([40, 200], [3, 70], 2, 128, 16, seed=1, front=5, behind=9).check(ctx, 4)
    Cache([40, 200], [1, 1], 2, 128, 16, seed=1, front=2, behind=3).check(ctx, 4)
    Cache([40, 200], [0, 0], 2, 128, 16, seed=1, front=2, behind=3).check(ctx, 4)


@pytest.mark.parametrize("value", [float("inf"), float("nan"), -float("inf")])
def test_keys_that_are_not_numbers_reach_only_who_sees_them(ctx, value):
    """Values of later tokens, and of tokens before the window, that are not finite."""
    for window, first in ((0, 0), (40, 3)):
        c = Cache([90, 300], [30, 200], 2, 128, 16, seed=3)
        for b, j in ((0, 75), (1, 150), (1, 299), (1, 60)):
            c.v[int(c.table[b, j // 16]), :, j % 16, 5] = value
        q = torch.randn(c.T, 8, 128, generator=c.g, device="cuda").to(BF16)
        out = c.attend(ctx, q, window, first)
        want = plain.attend(q, c.k, c.v, c.table, c.lens, c.starts, window, first, 128 ** -0.5)
        fine = want.isfinite()
        assert torch.equal(out.isfinite(), fine)  # a weight times infinity may come out as NaN: weights are sums of two terms, one of which may be 0
        assert ((out.double() - want).abs()[fine] < 2 * HALF * want.abs()[fine] + 1e-3).all()  # roundings are test_chunks' business
    c = Cache([90, 300], [30, 200], 2, 128, 16, seed=3)
    c.k[int(c.table[0, 4]), :, 11, 5] = value  # position 75 of sequence 0
    q = torch.randn(c.T, 8, 128, generator=c.g, device="cuda").to(BF16)
    out = c.attend(ctx, q)
    want = plain.attend(q, c.k, c.v, c.table, c.lens, c.starts, 0, 0, 128 ** -0.5)
    assert torch.equal(out[:15].isnan(), want[:15].isnan()) and not out[:15].isnan().any() and not out[30:].isnan().any()


def test_scores_of_minus_infinity(ctx):
    """A row all of whose scores are -inf gets zeros; one that sees such keys first and others later, the others."""
    for new in (1, 160):
        c = Cache([400], [new], 1, 128, 16, seed=new)
        for j in range(200):
            c.k[int(c.table[0, j // 16]), 0, j % 16] = 0
            c.k[int(c.table[0, j // 16]), 0, j % 16, 0] = -float("inf")
        q = torch.rand(c.T, 2, 128, generator=c.g, device="cuda").to(BF16) + 0.5
        c.compare(q, c.attend(ctx, q))
        c.compare(q, c.attend(ctx, q, 30, 40), 30, 40)
        c.k[:, :, :, 0], c.k[:, :, :, 1:] = -float("inf"), 0
        assert (c.attend(ctx, q) == 0).all()


@pytest.mark.parametrize("amp", [1e-3, 30.0])
def test_flat_and_peaked_scores(ctx, amp):
    Cache([700, 900], [1, 1], 2, 128, 64, seed=2).check(ctx, 4, amp=amp)
    Cache([700, 900], [5, 140], 2, 128, 64, seed=2).check(ctx, 4, amp=amp)


def test_maxima_that_grow(ctx):
    """Scores that rise along the keys by more than any lazy rescaling lets pass."""
    for new in (1, 40):
        c = Cache([1000], [new], 1, 64, 16, seed=4)
        for j in range(1000):
            c.k[int(c.table[0, j // 16]), 0, j % 16] = j / 100.0
        q = torch.full((c.T, 4, 64), 1.0, device="cuda").to(BF16)
        c.compare(q, c.attend(ctx, q))


@pytest.mark.parametrize("new", [1, 6, 300])
def test_long_sequences_in_parts(ctx, new):
    """Few rows over many keys: the keys are shared out and joined."""
    c = Cache([9000, 40, 5001], [new, min(new, 40), new], 1, 128, 32, seed=new)
    q = torch.randn(c.T, 4, 128, generator=c.g, device="cuda").to(BF16)
    out = c.attend(ctx, q)
    pick = [0, c.starts[1] - 1, c.starts[1], c.starts[2], c.T - 1]
    for i in pick:
        b = max(x for x in range(3) if c.starts[x] <= i)
        p = c.lens[b] - c.starts[b + 1] + i
        want, size, scores = plain.attend(q[i:i + 1], c.k, c.v, c.table[b:b + 1], [p + 1], [0, 1], 0, 0, 128 ** -0.5, True)
        bound = HALF * want.abs() + size * (2.0 ** -15 + 2 * scores * 130 * 2.0 ** -24 + 2 * 9000 * 2.0 ** -24)
        assert ((out[i].double() - want[0]).abs() <= bound[0] * (1 + HALF)).all(), i
    assert torch.equal(c.attend(ctx, q), out), "the same call twice"
    again = c.attend(ctx, q, max_len=100)  # it is for planning: sequences that are longer are computed too
    assert ((again.double() - out.double()).abs() <= 4 * HALF * out.double().abs() + 1e-4).all()


def test_caches_of_more_than_2_to_the_31_elements(ctx):
    Hkv, D, page = 8, 128, 256
    n_pages = 2 ** 31 // (Hkv * D * page) + 40
    k, v = (torch.zeros(n_pages, Hkv, page, D, dtype=BF16, device="cuda") for _ in range(2))
    for new in (1, 50):
        c = Cache([600, 300], [new, new], Hkv, D, page, seed=new)
        far = torch.tensor([n_pages - 1 - i for i in range(c.n_pages)], device="cuda")
        k[far], v[far] = c.k, c.v
        near, near_table = (c.k, c.v, c.n_pages), c.table
        c.table = torch.where(c.table >= 0, n_pages - 1 - c.table, c.table)
        q = torch.randn(c.T, 32, D, generator=c.g, device="cuda").to(BF16)
        c.k, c.v, c.n_pages = k, v, n_pages
        out = c.attend(ctx, q)
        (c.k, c.v, c.n_pages), c.table = near, near_table
        assert torch.equal(out, c.attend(ctx, q))
        qkv = torch.randn(c.T, (32 + 16) * D, generator=c.g, device="cuda").to(BF16)
        gain = torch.ones(D, device="cuda")
        qq = torch.zeros_like(q)
        torch.cuda.synchronize()
        for kk, vv, pages, table in ((k, v, n_pages, torch.where(c.table >= 0, n_pages - 1 - c.table, c.table)), (c.k, c.v, c.n_pages, c.table)):
            torch.cuda.synchronize()
            N.check(L().strictb200_rope_qknorm_paged(ctx.h, ptr(qkv), ptr(table), ptr(c.d_lens), ptr(c.d_starts), 2, c.T, 32, Hkv, D, ptr(gain), ptr(gain), 1e-6, 1e4,
                                                     pages, page, c.ld, ptr(qq), ptr(kk), ptr(vv)))
            ctx.synchronize()
        assert torch.equal(torch.nan_to_num(k[far]), torch.nan_to_num(c.k)) and torch.equal(torch.nan_to_num(v[far]), torch.nan_to_num(c.v))
    before = k[n_pages - 1].clone()
    src, dst = np.array([n_pages - 1], np.int32), np.array([n_pages - 35], np.int32)
    pools = np.array([k.data_ptr()], np.uint64)
    torch.cuda.synchronize()
    N.check(L().strictb200_pages_copy(ctx.h, N.ptr(pools), 1, n_pages, Hkv * page * D * 2, N.ptr(src), N.ptr(dst), 1))
    ctx.synchronize()
    assert torch.equal(torch.nan_to_num(k[n_pages - 35]), torch.nan_to_num(before))


@pytest.mark.parametrize("new", [1, 20])
def test_recorded_calls(ctx, new):
    """Two recorded sequences that share the context's scratch, replayed with other lengths than they were recorded with."""
    a, b = (Cache([2000, 900, 77], [new] * 3, 2, 128, 16, seed=s) for s in (1, 2))
    qs = [torch.randn(c.T, 8, 128, generator=c.g, device="cuda").to(BF16) for c in (a, b)]
    outs = [torch.full_like(q, 7.0) for q in qs]
    for c, q, o in zip((a, b), qs, outs):
        c.attend(ctx, q, out=o)  # scratch grows outside
    graphs = []
    for c, q, o in zip((a, b), qs, outs):
        with ctx.record():
            N.check(L().strictb200_attn_paged(ctx.h, ptr(q), ptr(c.k), ptr(c.v), ptr(c.table), ptr(c.d_lens), ptr(c.d_starts), 3, c.T, new, 2000, 8, 2, 128, c.n_pages,
                                              16, c.ld, 0, 0, 128 ** -0.5, ptr(o)))
        graphs.append(ctx.last_graph)
    a.lens, b.lens = [1500, 899, 60], [1999, 30, 77]
    for c, o in zip((a, b), outs):
        c.d_lens.copy_(torch.tensor(c.lens, dtype=torch.int32))
        o.fill_(7.0)
    torch.cuda.synchronize()
    for g in graphs:
        ctx.replay(g)
    ctx.synchronize()
    for c, q, o in zip((a, b), qs, outs):
        c.compare(q, o)
    for g in graphs:
        ctx.free_graph(g)


# ------------------------------------------------------------------ norm, rotation, append
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (12, 12, 64), (7, 1, 128), (1, 1, 64)])
@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("norm", [True, False])
def test_append(ctx, Hq, Hkv, D, page, norm):
    for lens, new, front, behind in (([1, 30, 300], [1, 1, 1], 0, 0), ([40, 0, 1, 513], [40, 0, 1, 200], 2, 3), ([7] * 40, [2] * 40, 0, 0)):
        c = Cache(lens, new, Hkv, D, page, seed=Hq, rest=0.0, front=front, behind=behind)
        qkv = torch.randn(c.T, (Hq + 2 * Hkv) * D, generator=c.g, device="cuda").to(BF16)
        gains = [1 + 0.3 * torch.randn(D, generator=c.g, device="cuda") for _ in range(2)] if norm else [None, None]
        q = torch.full((c.T, Hq, D), 7.0, dtype=BF16, device="cuda")
        want = plain.append(qkv, c.table, c.lens, c.starts, Hq, Hkv, D, *gains, 1e-6, 1e6, q, c.k, c.v)
        torch.cuda.synchronize()
        N.check(L().strictb200_rope_qknorm_paged(ctx.h, ptr(qkv), ptr(c.table), ptr(c.d_lens), ptr(c.d_starts), len(lens), c.T, Hq, Hkv, D, ptr(gains[0]),
                                                 ptr(gains[1]), 1e-6, 1e6, c.n_pages, page, c.ld, ptr(q), ptr(c.k), ptr(c.v)))
        ctx.synchronize()
        for got, w, pair in zip((q, c.k, c.v), want, (True, True, False)):
            # the output's rounding; the norm's D sums, its root and products (D + 8 roundings of 2^-24), and an angle that is off by 2^-24 turns, of a pair
            other = torch.cat([w[..., D // 2:], w[..., :D // 2]], -1).abs() if pair else 0
            bound = HALF * w.abs() + (w.abs() + other) * ((D + 8) * 2.0 ** -24 + 2 * np.pi * 2.0 ** -24)
            assert ((got.double() - w).abs() <= bound).all(), float(((got.double() - w).abs() - bound).max())


@pytest.mark.parametrize("pos", [100000, 2 ** 24 + 1, 2 ** 31 - 2])
def test_append_far_positions(ctx, pos):
    """Angles of positions that fp32 does not hold, and positions beyond the table (nothing is written)."""
    D, g = 128, torch.Generator("cuda").manual_seed(5)
    qkv = torch.randn(1, 3 * D, generator=g, device="cuda").to(BF16)
    k, v = (torch.zeros(2, 1, 16, D, dtype=BF16, device="cuda") for _ in range(2))
    q = torch.zeros(1, 1, D, dtype=BF16, device="cuda")
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    lens, starts = torch.tensor([pos + 1], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    want = plain.append(qkv, table, [pos + 1], [0, 1], 1, 1, D, None, None, 0.0, 1e4, q, k, v)
    torch.cuda.synchronize()
    N.check(L().strictb200_rope_qknorm_paged(ctx.h, ptr(qkv), ptr(table), ptr(lens), ptr(starts), 1, 1, 1, 1, D, None, None, 0.0, 1e4, 2, 16, 1, ptr(q), ptr(k), ptr(v)))
    ctx.synchronize()
    assert ((q.double() - want[0]).abs() <= HALF * want[0].abs() + 8 * 2 * np.pi * 2.0 ** -24).all()
    assert (k == 0).all() and (v == 0).all()


# ------------------------------------------------------------------ page copies
@pytest.mark.parametrize("pools,n_pages,page_bytes,n", [(1, 4, 16, 1), (3, 50, 4112, 20), (100, 40, 512, 11), (2, 2000, 64, 1000), (1, 3, 3 << 20, 1)])
def test_page_copies(ctx, pools, n_pages, page_bytes, n):
    rng = np.random.default_rng(n)
    data = [torch.randint(0, 256, (n_pages, page_bytes), dtype=torch.uint8, device="cuda") for _ in range(pools)]
    order = rng.permutation(n_pages).astype(np.int32)
    dst = order[:n].copy()
    src = rng.choice(order[n:], n).astype(np.int32)  # sources may come more than once
    want = [d.clone() for d in data]
    for w, d in zip(want, data):
        w[torch.from_numpy(dst).long().cuda()] = d[torch.from_numpy(src).long().cuda()]
    where = np.array([d.data_ptr() for d in data], np.uint64)
    torch.cuda.synchronize()
    N.check(L().strictb200_pages_copy(ctx.h, N.ptr(where), pools, n_pages, page_bytes, N.ptr(src), N.ptr(dst), n))
    src[:], dst[:] = 0, 0  # the call has read them
    ctx.synchronize()
    assert all(torch.equal(d, w) for d, w in zip(data, want))
