"""What the operators of a paged cache decide from sizes and wishes alone, at the ends of their ranges: the library's own functions, called on the host."""
import ctypes as C

import numpy as np
import pytest

from strict_b200 import native as N
from test_paged_cpu import A, attn, sample

ONE = 2.0 ** 43  # the weight of the largest logit


def reach(total, want, n, heat, top):
    f = N.lib()._Z13sb_draw_reachmmiff
    f.restype, f.argtypes = C.c_float, [C.c_uint64, C.c_uint64, C.c_int, C.c_float, C.c_float]
    return np.float32(f(total, want, n, heat, top))


def wanted(total, top_p):
    """top_p of a sum of whole numbers, rounded up, at least 1."""
    num, den = float(top_p).as_integer_ratio()
    return max(1, -(-total * num // den))


def held(x, heat, top_p):
    """The sum of a row's weights, what top_p wants of it, and what the logits within reach hold."""
    x = np.asarray(x, np.float32)
    w = np.rint(np.exp((x.astype(np.float64) - float(x.max())) / float(np.float32(heat))) * ONE).astype(np.uint64)
    total = int(w.sum())
    want = wanted(total, np.float32(top_p))
    low = x.max() - reach(total, want, len(x), heat, x.max())
    return total, want, int(w[x >= low].sum())


@pytest.mark.parametrize("n,top,rest,top_p", [(151936, 0.0, -27.918, 0.9999999), (144000, 28.5468, 0.0, 1 - 2.0 ** -24)])
def test_bins_hold_what_top_p_wants_over_a_flat_tail(n, top, rest, top_p):
    """Weights of the tail round up: 6.6 to 7, 3.52 to 4."""
    x = np.full(n, rest, np.float32)
    x[n // 3] = top
    total, want, there = held(x, 1.0, top_p)
    assert total > ONE and there >= want


def test_bins_hold_what_top_p_wants():
    """Any tail, around the logits that weigh a whole number and a half, and any heat and place of the largest logit."""
    rng = np.random.default_rng(5)
    for i in range(600):
        many, peaks = i % 4 == 0, int(rng.integers(1, 4))
        n = int(2 ** (rng.uniform(15, 20) if many else rng.uniform(1, 14)))
        heat, top = np.float32(10 ** rng.uniform(-4, 8)), np.float32(rng.choice([0.0, 0.0, 1.0, -7.5, 1e4]))
        # many: as a share of the rest that one of the larger top_p leaves out
        whole = int(ONE * peaks * 2.0 ** -24 * rng.integers(1, 13) / n) if many else int(10 ** rng.uniform(0, 12.9))
        # weights a little above whole + 1/2, or spread over some more
        x = float(top) + float(heat) * np.log((whole + 0.5 + rng.uniform(0.001, 1, n) * rng.choice([1e-2, 1, 30])) / ONE)
        x = np.minimum(x, float(top)).astype(np.float32)
        x[rng.choice(n, min(n, peaks), replace=False)] = top
        for top_p in [1 - 2.0 ** -24 * j for j in range(1, 13)] + [0.999, 0.9, 0.5, 1e-3, 0.0]:
            total, want, there = held(x, heat, top_p)
            assert there >= want, (i, n, heat, top, whole, top_p)


@pytest.mark.parametrize("n", [2, 1000, 2 ** 20])
def test_bins_hold_what_top_p_wants_of_equal_logits(n):
    for top_p in (0.0, 2.0 ** -149, 1e-7, 0.5, 1 - 2.0 ** -24):
        for down in (0.0, 1e-13, 1e-12, 1e-6):
            x = np.full(n, -down, np.float32)
            x[0] = 0.0
            total, want, there = held(x, 1.0, top_p)
            assert there >= want


def test_an_infinite_heat_leaves_nothing_out():
    assert not reach(2 ** 43 * 10, 2 ** 43 * 3, 10, float("inf"), 1.0) < 1e30


@pytest.mark.parametrize("wish,n,k,lists", [(0, 10, 0, False), (-1, 10, 0, False), (-2 ** 31, 10, 0, False), (1, 1, 0, False), (1, 2, 1, True), (9, 10, 9, True), (10, 10, 0, False),
                                            (11, 10, 0, False), (256, 1000, 256, True), (257, 1000, 257, False), (256, 256, 0, False), (2 ** 20 - 1, 2 ** 20, 2 ** 20 - 1, False),
                                            (2 ** 30, 2 ** 20, 0, False), (2 ** 30 + 1, 2 ** 20, 0, False), (2 ** 31 - 1, 2 ** 20, 0, False)])
def test_top_k_of_every_size(wish, n, k, lists):
    """Off below 1 and from the number of tokens on, however large; a list is tried for up to 256."""
    cut, tried = N.lib()._Z13sb_draw_top_kii, N.lib()._Z13sb_draw_listsi
    cut.restype, cut.argtypes, tried.restype, tried.argtypes = C.c_int, [C.c_int, C.c_int], C.c_bool, [C.c_int]
    assert cut(wish, n) == k and tried(k) == lists


FAR = A + 2 ** 40
ROWS, PAGES = 2 * 8 * 128 * 2, 4 * 2 * 16 * 128 * 2  # bytes of the rows and of the pages of attn()'s arguments


@pytest.mark.parametrize("out", [A + 16, A - 16, A + ROWS - 16, A - ROWS + 16])
def test_attention_refuses_rows_over_other_rows_queries(out):
    with pytest.raises(ValueError, match="out overlaps q"):
        attn(k=FAR, v=FAR, out=out)


@pytest.mark.parametrize("name", ["k", "v"])
@pytest.mark.parametrize("out", [A, A + PAGES - 16, A - ROWS + 16])
def test_attention_refuses_rows_over_pages(name, out):
    with pytest.raises(ValueError, match="pages"):
        attn(**{"q": FAR, "k": FAR, "v": FAR, name: A}, out=out)


@pytest.mark.parametrize("kw", [dict(out=A), dict(out=A + 4 * 249), dict(out=A - 4), dict(out=FAR, prob=A + 4 * 249), dict(out=FAR, prob=FAR), dict(out=FAR, prob=FAR + 4),
                                dict(out=A + 2 * 248, dtype=0)], ids=str)
def test_draws_refuse_results_over_logits(kw):
    """Two rows of 100 logits, 150 apart."""
    with pytest.raises(ValueError, match="overlap"):
        sample(**{**dict(M=2, N=100, ld=150, u=FAR, t=FAR, k=FAR, p=FAR, q=FAR, prob=None), **kw})
