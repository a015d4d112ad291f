"""The operators of a paged cache at the ends of what they take (plain forms: paged_plain.py)."""
import time

import numpy as np
import pytest
import torch

import paged_plain as plain
from strict_b200 import native as N
from test_gpu_draw import check, logits, sample
from test_gpu_paged import Cache

pytestmark = pytest.mark.gpu
ONE = 2.0 ** 43


def draw_whole(x, u, heat, top_k, top_p, min_p):
    """Token and share of a row whose weights are whole numbers, 2^43 for the largest logit, in exact arithmetic."""
    x = np.asarray(x, np.float32).astype(np.float64)
    top = x.max()
    w = np.where(x == top, ONE, 0.0) if top == np.inf else np.rint(np.exp((x - top) / heat) * ONE)  # beside infinity nothing weighs anything
    w = w.astype(np.uint64)
    order = np.lexsort((np.arange(len(x)), -x))
    keep = order[:top_k] if 0 < top_k < len(x) else order
    sums = np.cumsum(w[keep])
    if top_p < 1:
        num, den = float(top_p).as_integer_ratio()
        want = max(1, -(-int(sums[-1]) * num // den))
        keep = keep[:int(np.searchsorted(sums, np.uint64(want), side="left")) + 1]
    if min_p > 0:
        keep = keep[w[keep] >= np.uint64(np.ceil(min(min_p, 1.0) * ONE))]
    keep = np.sort(keep)
    sums = np.cumsum(w[keep])
    num, den = float(u).as_integer_ratio()
    at = int(np.searchsorted(sums, np.uint64(int(sums[-1]) * num // den), side="right"))
    return int(keep[at]), float(w[keep[at]]) / float(sums[-1])


def check_whole(ctx, x, u, heat=1.0, top_k=0, top_p=1.0, min_p=0.0, off=0.0):
    """off: by how much a weight may differ, in units of the largest."""
    M = x.shape[0]
    rows = [np.broadcast_to(np.asarray(v, t), (M,)) for v, t in ((u, np.float32), (heat, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32))]
    got, prob = sample(ctx, x, rows[0], temperature=rows[1], top_k=rows[2], top_p=rows[3], min_p=rows[4])
    host = x.float().cpu().numpy()
    for m in range(M):
        token, share = draw_whole(host[m], *[r[m].item() for r in rows])
        # the quotient of two whole numbers, rounded to fp32 (by way of fp64)
        assert got[m] == token and abs(float(prob[m]) - share) <= 2.0 ** -24 * (1 + 1e-6) * share + x.shape[1] * off, (m, got[m], token, prob[m], share)


# Weights of the tail (6.6, 3.52, ..) are far enough from a half that every way to compute them rounds them alike.
TAILS = [(151936, 6.6), (144000, 3.52), (50257, 10.8), (2 ** 20, 0.7), (20011, 26.3)]


@pytest.mark.parametrize("peaks", [1, 3, 700])
@pytest.mark.parametrize("n,weight", TAILS)
@pytest.mark.parametrize("rows", [1, 5, 200])
def test_top_p_next_to_one_over_a_flat_tail(ctx, n, weight, rows, peaks):
    """Logits whose weights are rounded up to more than what top_p leaves out gives to each of them."""
    if rows * n > 5_000_000:
        rows = 3
    for top, heat in ((0.0, 1.0), (28.5468, 0.7)):
        x = torch.full((rows, n), float(np.float32(top + heat * np.log(weight / ONE))), device="cuda")
        at = np.random.default_rng(n).choice(n, peaks, replace=False)
        x[:, at] = top
        u = np.linspace(0, 1 - 2.0 ** -24, rows).astype(np.float32)
        for top_p in (1 - 2.0 ** -24, 1 - 2.0 ** -23, 0.9999999, 0.999999):
            check_whole(ctx, x[:, :], u, heat, 0, top_p)
        check_whole(ctx, x, u, heat, max(peaks + 1, n // 2), 1 - 2.0 ** -24)


@pytest.mark.parametrize("rows", [5, 200])
@pytest.mark.parametrize("top_k", [2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1, -2 ** 31])
def test_top_k_beyond_every_row(ctx, rows, top_k):
    """It is off, beside a top_p too, for few rows and for many."""
    x, u = logits(rows, 20011, rows), np.random.default_rng(3).random(rows, np.float32)
    for kw in (dict(top_p=0.9), dict(top_p=0.3, min_p=0.01), dict(top_p=0.95, temperature=3.0)):
        got, want = sample(ctx, x, u, top_k=top_k, **kw), sample(ctx, x, u, **kw)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    check(ctx, x[:5], u[:5], top_k=top_k, top_p=0.9)


@pytest.mark.parametrize("heat", [1e-30, 1e-37, 1.2e-38, 1e-40, 1e-45])
def test_heats_among_the_least_numbers(ctx, heat):
    """Logits as near to one another as such heats are small: 0, subnormal numbers, the least normal ones."""
    tiny = float(np.finfo(np.float32).tiny)
    rows = []
    for top in (0.0, -0.0, tiny, tiny / 8, -tiny / 4):
        x = np.full(3000, -1.0, np.float32)
        x[[5, 700, 2999]] = top
        x[::7] = np.float32(top - heat)
        x[[1, 9]] = np.float32(top - 3 * heat)
        rows.append(x)
    x = torch.from_numpy(np.stack(rows)).cuda()
    for u in (0.0, 0.5, 0.99):
        for kw in (dict(), dict(top_p=0.9), dict(top_p=0.999999, top_k=900), dict(min_p=0.1), dict(top_k=2)):
            # running sums may meet their targets exactly, so by whole numbers: equal logits have equal ones, off by one at most
            check_whole(ctx, x, u, heat, **kw, off=2.0 ** -43)


@pytest.mark.parametrize("heat", [1e36, 1e38, float("inf")])
@pytest.mark.parametrize("rows", [2, 150])
def test_heats_without_an_end(ctx, heat, rows):
    """Everything weighs the same; beside infinities nothing else does."""
    n = 20011
    x = logits(rows, n, 3)
    u = np.linspace(0, 1 - 2.0 ** -24, rows).astype(np.float32)
    some = torch.randperm(n, generator=torch.Generator("cuda").manual_seed(1), device="cuda")[:1000]
    for fill in (None, float("inf"), torch.finfo(torch.float32).max):
        if fill is not None:
            x[:, some] = fill
        for kw in (dict(), dict(top_k=300), dict(top_k=999), dict(top_k=1000), dict(top_k=1001), dict(top_p=0.25), dict(top_k=700, top_p=0.5), dict(top_k=2000, top_p=0.9)):
            if rows > 2 and len(kw) != 1:
                continue
            check_whole(ctx, x, u, heat, **kw, off=2.0 ** -43)  # weights below 2^-44 of the largest are 0, the others here are all the same


@pytest.mark.parametrize("m", [3, 400])
def test_results_over_what_a_row_reads_once(ctx, m):
    """Tokens over the random numbers, shares over min_p."""
    n = 20011
    rng = np.random.default_rng(6)
    x, u, least = logits(m, n, 6), rng.random(m, np.float32), rng.choice([0.0, 0.05, 0.3], m).astype(np.float32)
    k, p = rng.choice([0, 3, 5000], m).astype(np.int32), rng.choice([0.5, 0.9, 1.0], m).astype(np.float32)
    want = sample(ctx, x, u, top_k=k, top_p=p, min_p=least)
    du, dk, dp, dq = (torch.from_numpy(v).cuda() for v in (u, k, p, least))
    torch.cuda.synchronize()
    N.check(N.lib().strictb200_sample(ctx.h, x.data_ptr(), 1, m, n, n, du.data_ptr(), None, dk.data_ptr(), dp.data_ptr(), dq.data_ptr(), du.data_ptr(), dq.data_ptr()))
    ctx.synchronize()
    assert np.array_equal(du.cpu().numpy().view(np.int32), want[0]) and np.array_equal(dq.cpu().numpy(), want[1])


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("new,G,D", [(1, 4, 128), (4, 4, 64), (20, 4, 128), (200, 4, 64), (150, 5, 128)])
@pytest.mark.parametrize("lens", [[7000, 300, 40], [260, 700] * 15])
def test_rows_in_place_of_their_queries(ctx, new, G, D, lens):
    """Every way the keys are cut and joined."""
    c = Cache([max(n, new) for n in lens], [new] * len(lens), 2, D, 16, seed=new, front=1, behind=2)
    q = torch.randn(c.T, 2 * G, D, generator=c.g, device="cuda").to(torch.bfloat16)
    q[0], q[-2:] = 7.0, 7.0
    want = c.attend(ctx, q)
    for _ in range(3):
        own = q.clone()
        assert torch.equal(c.attend(ctx, own, out=own), want)


def attend_far(ctx, c, q, far, window=0, first=0, max_len=None):
    """Sequence `far` is as long as an int32 says; what lies in the table is all that there is to see. Compared with a length just behind the table."""
    c.d_lens[far] = 2 ** 31 - 1
    out = c.attend(ctx, q, window, first, max_len=max_len)
    c.lens[far] = c.ld * c.page + c.starts[far + 1] - c.starts[far]
    c.compare(q, out, window, first)


@pytest.mark.parametrize("new,G,far", [(1, 4, 0), (3, 4, 2), (12, 4, 0), (30, 4, 5), (100, 4, 0), (100, 4, 19), (150, 2, 7), (300, 1, 0)])
@pytest.mark.parametrize("max_len", [None, 5000])
def test_a_length_without_an_end(ctx, new, G, far, max_len):
    """More units than SMs, so that each is searched for: the others' rows are there too."""
    rng = np.random.default_rng(new)
    lens = [int(x) + new for x in rng.integers(1, 500, 20)]
    lens[far] = new + 700
    c = Cache(lens, [new] * 20, 8, 64, 32, seed=new)
    q = torch.randn(c.T, 8 * G, 64, generator=c.g, device="cuda").to(torch.bfloat16)
    attend_far(ctx, c, q, far, max_len=max_len)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 20, 2 ** 30 + 5])
@pytest.mark.parametrize("lens,new", [([3, 40], [5, 9]), ([3, 40], [4, 1]), ([100, 500], [150, 30]), ([60, 3, 200], [70, 9, 200])])
def test_windows_that_hide_nothing(ctx, window, lens, new):
    """As wide as an int32 says, rows in front of their sequence among the new ones, and values that are not finite."""
    for first in (0, 7, 2 ** 31 - 1):
        c = Cache(lens, new, 2, 64, 16, seed=3)
        q, out = c.check(ctx, 2, window, first)
        assert torch.equal(out, c.attend(ctx, q))
    c.v[int(c.table[0, 0]), :, 2, 5] = float("nan")
    out = c.attend(ctx, q, window)
    want = plain.attend(q, c.k, c.v, c.table, c.lens, c.starts, 0, 0, 64 ** -0.5)
    assert torch.equal(out.isnan(), want.isnan())


def milliseconds(ctx, call, n=5):
    """The least of n calls, by the host's clock around calls that are waited for."""
    best = 1e9
    for _ in range(n):
        ctx.synchronize()
        t = time.perf_counter()
        call()
        ctx.synchronize()
        best = min(best, (time.perf_counter() - t) * 1e3)
    return best


@pytest.mark.parametrize("new,D", [(1, 128), (6, 64), (25, 128), (200, 128)])
def test_one_nan_does_not_hold_up_a_long_sequence(ctx, new, D):
    """Values that are not finite, in tiles that some row does not see, are looked up again in those tiles only, however long the sequence is."""
    lens = [16000 + new, 300 + new, 500 + new]
    c = Cache(lens, [new] * 3, 2, D, 16, seed=new)
    q = torch.randn(c.T, 8, D, generator=c.g, device="cuda").to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    call = lambda: c.attend(ctx, q, out=out)  # noqa: E731
    call()
    before, fine = milliseconds(ctx, call), out.clone()
    c.v[int(c.table[0, (lens[0] - 1) // 16]), :, (lens[0] - 1) % 16, 9] = float("nan")  # the last position: only the last row sees it
    c.v[int(c.table[0, 3]), :, 5, 11] = -float("inf")  # all rows see this one
    after = milliseconds(ctx, call)
    last = c.starts[1] - 1
    assert out[last, :, 9].isnan().all() and not out[:c.starts[1], :, 11].isfinite().any()
    same = torch.ones_like(q, dtype=torch.bool)
    same[last, :, 9], same[:c.starts[1], :, 11] = False, False
    assert torch.equal(out[same], fine[same])
    assert after < 2 * before + 0.3, (before, after)


@pytest.mark.parametrize("new,G,D", [(1, 4, 64), (5, 3, 128), (25, 4, 64), (90, 4, 128), (400, 2, 64)])
@pytest.mark.parametrize("window,first", [(0, 0), (900, 300)])
def test_values_that_are_not_finite_between_pages_that_are_missing(ctx, new, G, D, window, first):
    """Many tiles that no row sees whole, each with such values in a dim of its own: more of them than a block takes down, and few."""
    for every in (1, 9):
        c = Cache([3000, 700], [new, new], 2, D, 16, seed=new + every)
        q = torch.randn(c.T, 2 * G, D, generator=c.g, device="cuda").to(torch.bfloat16)
        for b in (0, 1):
            for i in range(0, c.lens[b] // 16 - 4, 5):
                c.table[b, i + 1] = -1
                if i // 5 % every == 0:
                    c.v[int(c.table[b, i]), :, i % 16, i // 5 % D] = float("nan") if i % 2 else float("inf")
            c.v[int(c.table[b, (c.lens[b] - 1) // 16]), :, (c.lens[b] - 1) % 16, D - 1] = float("nan")
        out = c.attend(ctx, q, window, first)
        want = plain.attend(q, c.k, c.v, c.table, c.lens, c.starts, window, first, D ** -0.5)
        assert torch.equal(out.isfinite(), want.isfinite())
        fine = want.isfinite()
        assert ((out.double() - want).abs()[fine] < 2 * torch.finfo(torch.bfloat16).eps * want.abs()[fine] + 1e-3).all()  # roundings are test_chunks' business
