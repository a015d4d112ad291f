"""strictb200_sample against its definition in 64 bits (paged_plain.draw): the same token in every row, its share to fp32."""
import numpy as np
import pytest
import torch

import paged_plain as plain
from strict_b200 import native as N

pytestmark = pytest.mark.gpu


def sample(ctx, x, u, temperature=None, top_k=None, top_p=None, min_p=None, ld=None, want_prob=True):
    M, n = x.shape
    dev = lambda v, t: None if v is None else torch.as_tensor(np.broadcast_to(np.asarray(v), (M,)).copy()).to(t).cuda()  # noqa: E731
    args = [dev(u, torch.float32), dev(temperature, torch.float32), dev(top_k, torch.int32), dev(top_p, torch.float32), dev(min_p, torch.float32)]
    out, prob = torch.full((M,), -9, dtype=torch.int32, device="cuda"), torch.full((M,), -9.0, device="cuda")
    torch.cuda.synchronize()
    N.check(N.lib().strictb200_sample(ctx.h, x.data_ptr(), 1 if x.dtype == torch.float32 else 0, M, n, ld or x.stride(0) or n,
                                      *[None if a is None else a.data_ptr() for a in args], out.data_ptr(), prob.data_ptr() if want_prob else None))
    ctx.synchronize()
    return out.cpu().numpy(), prob.cpu().numpy()


def check(ctx, x, u, temperature=None, top_k=None, top_p=None, min_p=None):
    M = x.shape[0]
    got, prob = sample(ctx, x, u, temperature, top_k, top_p, min_p)
    rows = lambda v, off, t: np.broadcast_to(np.asarray(off if v is None else v, t), (M,))  # noqa: E731
    host = x.float().cpu().numpy()
    for m, (uu, t, k, p, q) in enumerate(zip(rows(u, 0, np.float32), rows(temperature, 1, np.float32), rows(top_k, 0, np.int32), rows(top_p, 1, np.float32),
                                             rows(min_p, 0, np.float32))):
        token, share = plain.draw(host[m], float(uu), float(t), int(k), float(p), float(q))
        # fp32 rounding of a quotient of weights that are off by 2^-42 of the largest each (the difference in 64 bits: of fp32 values it would be rounded itself)
        assert got[m] == token and abs(float(prob[m]) - share) <= 2.0 ** -24 * share + x.shape[1] * 2.0 ** -43, (m, got[m], token, prob[m], share)


def logits(M, n, seed, scale=3.0, dtype=torch.float32):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(M, n, generator=g, device="cuda") * scale).to(dtype)


SIZES = [1, 2, 31, 33, 1000, 1025, 5003, 50257, 151936]


@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("filters", [{}, dict(top_k=20), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=50, top_p=0.95), dict(top_k=700, top_p=0.5, min_p=0.1),
                                     dict(temperature=0.3, top_p=0.99), dict(temperature=5.0, top_p=0.99), dict(temperature=2.0, top_k=3000)], ids=str)
def test_draws(ctx, n, dtype, filters):
    x = logits(6, n, n, dtype=dtype)
    check(ctx, x, np.array([0.0, 0.1, 0.37, 0.5, 0.9, 0.99999], np.float32), **filters)


def test_every_row_its_own_wishes(ctx):
    M = 97
    rng = np.random.default_rng(3)
    x = logits(M, 4099, 5)
    off = lambda v, o: np.where(rng.random(M) < 0.4, o, v)  # noqa: E731
    check(ctx, x, rng.random(M, np.float32), off(rng.uniform(0.2, 3, M), 0.0).astype(np.float32), off(rng.integers(1, 5000, M), 0).astype(np.int32),
          off(rng.random(M), 1.0).astype(np.float32), off(rng.random(M) * 0.3, 0.0).astype(np.float32))


@pytest.mark.parametrize("n", [7, 3001, 151936])
def test_equal_logits(ctx, n):
    """Ties: the lower index is first, and sums meet the thresholds exactly."""
    x = torch.full((4, n), -1.5, device="cuda")
    u = np.array([0.0, 0.25, 0.5, 0.999], np.float32)
    check(ctx, x, u)
    check(ctx, x, u, top_k=3)
    check(ctx, x, u, top_k=n - 1)
    check(ctx, x, u, top_p=0.5)
    check(ctx, x, u, top_p=0.25, min_p=1.0)
    check(ctx, x, u, temperature=0.0)
    x[:, n // 2] = 2.0
    check(ctx, x, u, top_k=2, min_p=0.01)
    check(ctx, x, u, temperature=0.0)
    check(ctx, torch.round(logits(4, n, 9)), u, top_k=n // 3 + 1, top_p=0.7)


def test_values_that_are_not_numbers(ctx):
    n, inf, nan = 2000, float("inf"), float("nan")
    base = logits(1, n, 1)[0]
    rows = []
    for fill, at in ((-inf, slice(0, 1990)), (nan, slice(5, n)), (inf, slice(100, 102)), (-inf, slice(0, n)), (nan, slice(0, n)), (torch.finfo(torch.float32).min, slice(0, n)),
                     (torch.finfo(torch.float32).min, slice(0, 1500)), (torch.finfo(torch.float32).max, slice(3, 4))):
        r = base.clone()
        r[at] = fill
        rows.append(r)
    z = base.clone()
    z[:] = -5.0
    z[10], z[11] = -0.0, 0.0  # equal
    x = torch.stack(rows + [z])
    for u in (0.0, 0.3, 0.9):
        for filters in ({}, dict(top_k=2), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=0.0), dict(top_k=1500, top_p=0.99), dict(temperature=float("inf"))):
            check(ctx, x, u, **filters)


def test_parameters_at_their_ends(ctx):
    x = logits(8, 999, 2)
    for top_p in (0.0, -1.0, 1e-30, 1.0, 2.0, float("nan")):
        check(ctx, x, 0.4, top_p=top_p if top_p == top_p else 1.0)
        assert np.array_equal(sample(ctx, x, 0.4, top_p=top_p)[0], sample(ctx, x, 0.4, top_p=top_p if top_p == top_p else 1.0)[0])
    for min_p in (-1.0, 0.0, 1.0, 3.0):
        check(ctx, x, 0.4, min_p=min_p)
    for k in (-5, 0, 1, 998, 999, 1000, 2 ** 31 - 1):
        check(ctx, x, 0.4, top_k=k)
    for u in (-1.0, 1.0, 5.0, float("inf"), 1 - 2.0 ** -24, 1e-30):
        check(ctx, x, u)
    for t in (-1.0, 1e-30, 1e30):
        check(ctx, x, 0.4, temperature=t)
    assert np.array_equal(sample(ctx, x, float("nan"))[0], sample(ctx, x, 0.0)[0])
    assert np.array_equal(sample(ctx, x, 0.4, temperature=float("nan"))[0], sample(ctx, x, 0.4, temperature=0.0)[0])
    assert np.array_equal(sample(ctx, x, 0.4, min_p=float("nan"))[0], sample(ctx, x, 0.4)[0])


def test_rows_with_a_stride(ctx):
    for dtype, lead in ((torch.float32, 1), (torch.bfloat16, 3)):
        wide = logits(9, 1500, 3, dtype=dtype)
        view = wide[:, lead:lead + 1337]
        check(ctx, view, 0.6, top_k=40, top_p=0.9)
    got, prob = sample(ctx, view, 0.6, want_prob=False)
    assert (prob == -9).all()


def test_largest_vocabulary(ctx):
    x = logits(2, 1 << 20, 4)
    check(ctx, x, [0.3, 0.999], top_p=0.9)
    check(ctx, x, [0.3, 0.999], temperature=50.0)
    check(ctx, torch.zeros(1, 1 << 20, device="cuda"), 0.75, top_p=0.99)


def test_many_rows(ctx):
    x = logits(1000, 130, 6)
    check(ctx, x, np.random.default_rng(0).random(1000, np.float32), top_k=20, top_p=0.9, min_p=0.01)


def test_recorded(ctx):
    x = logits(3, 151936, 8)
    u = torch.tensor([0.2, 0.5, 0.8], device="cuda")
    p = torch.full((3,), 0.9, device="cuda")
    out = torch.zeros(3, dtype=torch.int32, device="cuda")
    call = lambda: N.check(N.lib().strictb200_sample(ctx.h, x.data_ptr(), 1, 3, 151936, 151936, u.data_ptr(), None, None, p.data_ptr(), None, out.data_ptr(), None))  # noqa: E731
    torch.cuda.synchronize()
    call()
    with ctx.record():
        call()
    x.copy_(logits(3, 151936, 9))
    torch.cuda.synchronize()
    ctx.replay(ctx.last_graph, 2)
    ctx.synchronize()
    ctx.free_graph(ctx.last_graph)
    assert out.tolist() == [plain.draw(x[m].cpu().numpy(), float(u[m]), 1.0, 0, float(p[m]), 0.0)[0] for m in range(3)]


@pytest.mark.parametrize("n", [1000, 20000, 60000])
@pytest.mark.parametrize("at", [0.0, 1e6, -1e4])
def test_cuts_at_the_end_of_many_equal_ones(ctx, n, at):
    """A bin of more equal logits than a list holds is kept to its last, and a little further down a few more begin."""
    rows = []
    for few in (1, 2, 3):
        x = torch.full((n,), at, dtype=torch.float32, device="cuda")
        x[7], x[n // 2 : n // 2 + few], x[11] = at + 0.0625, at - 0.0625, at + 0.0625
        rows += [x, x, x]
    x = torch.stack(rows)
    k = [v for few in (1, 2, 3) for v in (n - 1, n - few, n - few - 1)]
    check(ctx, x, 0.999, temperature=0.7, top_k=np.array(k, np.int32))
    check(ctx, x, 0.3, temperature=0.7, top_k=np.array(k, np.int32), top_p=0.5)
    w = np.exp(-0.0625 / 0.7)  # what the largest and the many hold of the weight, and a little less
    share = [(2 + (n - few - 2) * w - d) / (2 + (n - few - 2) * w + few * w * w) for few in (1, 2, 3) for d in (0.25, 0.75, 1.25)]
    check(ctx, x, 0.999, temperature=0.7, top_p=np.array(share, np.float32))


@pytest.mark.parametrize("m", [160, 1024, 1030])
def test_many_rows_of_different_length(ctx, m):
    """More rows than SMs, each its own block: the ones with a long way come first."""
    rng = np.random.default_rng(m)
    pick = lambda *v: np.array(rng.choice(v, m))  # noqa: E731
    check(ctx, logits(m, 20000, m), rng.random(m, np.float32), temperature=pick(0.0, 0.7, 1.0, 2.0).astype(np.float32), top_k=pick(0, 3, 300, 5000).astype(np.int32),
          top_p=pick(0.5, 0.9, 1.0).astype(np.float32), min_p=pick(0.0, 0.01).astype(np.float32))


@pytest.mark.parametrize("m", [3, 400])
def test_results_over_wishes(ctx, m):
    """Tokens may be written over top_k, shares over top_p or the temperature: a row's wishes are read before its results are written."""
    n = 20000
    rng = np.random.default_rng(5)
    x, u = logits(m, n, 5), torch.from_numpy(rng.random(m, np.float32)).cuda()
    t, k, p = rng.choice([0.0, 1.0], m).astype(np.float32), rng.choice([0, 3, 300, 5000], m).astype(np.int32), rng.choice([0.5, 0.9, 1.0], m).astype(np.float32)
    want = sample(ctx, x, u.cpu().numpy(), temperature=t, top_k=k, top_p=p)
    for over_p in (True, False):
        dt, dk, dp = (torch.from_numpy(v).cuda() for v in (t, k, p))
        prob = dp if over_p else dt
        torch.cuda.synchronize()
        N.check(N.lib().strictb200_sample(ctx.h, x.data_ptr(), 1, m, n, n, u.data_ptr(), dt.data_ptr(), dk.data_ptr(), dp.data_ptr(), None, dk.data_ptr(), prob.data_ptr()))
        ctx.synchronize()
        assert np.array_equal(dk.cpu().numpy(), want[0]) and np.array_equal(prob.cpu().numpy(), want[1])
