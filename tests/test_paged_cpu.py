"""Refusals of the operators of a paged cache and of the draw: the arguments are looked at before the context, so none of this needs a GPU. The context
handed in is an address that a refused call does not follow."""
import numpy as np
import pytest

from strict_b200 import native as N

CTX, A = 0x1000, 0x10000  # somewhere; 16-byte aligned


def attn(**kw):
    a = dict(ctx=CTX, q=A, k=A, v=A, table=A, lens=A, starts=A, B=2, T=2, max_new=1, max_len=10, Hq=8, Hkv=2, D=128, n_pages=4, page=16, ld=3, window=0, first=0,
             scale=0.1, out=A)
    a.update(kw)
    N.check(N.lib().strictb200_attn_paged(*a.values()))


def rope(**kw):
    a = dict(ctx=CTX, qkv=A, table=A, lens=A, starts=A, B=2, T=2, Hq=8, Hkv=2, D=128, qgain=A, kgain=A, eps=1e-6, theta=1e4, n_pages=4, page=16, ld=3, q=A, k=A, v=A)
    a.update(kw)
    N.check(N.lib().strictb200_rope_qknorm_paged(*a.values()))


def copy(src, dst, pools=(A,), n_pages=10, page_bytes=64, ctx=CTX):
    s, d, p = np.array(src, np.int32), np.array(dst, np.int32), np.array(pools, np.uint64)
    N.check(N.lib().strictb200_pages_copy(ctx, N.ptr(p) if len(p) else None, len(p), n_pages, page_bytes, N.ptr(s), N.ptr(d), len(s)))


def sample(**kw):
    a = dict(ctx=CTX, x=A, dtype=1, M=1, N=100, ld=100, u=A, t=A, k=A, p=A, q=A, out=A, prob=A)
    a.update(kw)
    N.check(N.lib().strictb200_sample(*a.values()))


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("kw", [dict(ctx=None), dict(B=-1), dict(T=-1), dict(max_new=-1), dict(max_len=-1), dict(Hq=0), dict(Hkv=0), dict(Hq=7), dict(Hq=-8), dict(n_pages=0),
                                dict(ld=0), dict(window=-1), dict(first=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=NAN), dict(scale=INF), dict(q=None), dict(k=None),
                                dict(v=None), dict(table=None), dict(lens=None), dict(starts=None), dict(out=None), dict(q=A + 2), dict(k=A + 8), dict(v=A + 4),
                                dict(out=A + 2), dict(T=2 ** 31)], ids=str)
def test_attention_refuses(kw):
    with pytest.raises(ValueError):
        attn(**kw)


@pytest.mark.parametrize("kw", [dict(D=96), dict(D=0), dict(page=8), dict(page=24), dict(page=512), dict(page=0), dict(page=-16), dict(Hq=129, Hkv=1), dict(Hq=65536, Hkv=1024),
                                dict(n_pages=2 ** 30, Hkv=8)], ids=str)
def test_attention_does_not_support(kw):
    with pytest.raises(NotImplementedError):
        attn(**kw)


@pytest.mark.parametrize("kw", [dict(ctx=None), dict(B=-1), dict(T=-1), dict(Hq=0), dict(Hkv=0), dict(n_pages=0), dict(ld=0), dict(theta=0.0), dict(theta=-1.0), dict(theta=NAN),
                                dict(theta=INF), dict(eps=-1.0), dict(eps=NAN), dict(qkv=None), dict(table=None), dict(lens=None), dict(starts=None), dict(q=None),
                                dict(k=None), dict(v=None), dict(qgain=None), dict(kgain=None), dict(qkv=A + 2), dict(q=A + 2), dict(k=A + 2), dict(v=A + 2),
                                dict(qgain=A + 4), dict(kgain=A + 4)], ids=str)
def test_append_refuses(kw):
    with pytest.raises(ValueError):
        rope(**kw)


@pytest.mark.parametrize("kw", [dict(D=32), dict(page=4), dict(page=48), dict(page=1024), dict(Hq=70000), dict(n_pages=2 ** 30, Hkv=8)], ids=str)
def test_append_does_not_support(kw):
    with pytest.raises(NotImplementedError):
        rope(**kw)


@pytest.mark.parametrize("args,kw", [(([1], [10]), {}), (([10], [1]), {}), (([-1], [1]), {}), (([1], [-1]), {}), (([1, 2], [3, 3]), {}), (([1, 3], [3, 4]), {}), (([1], [1]), {}),
                                     (([4, 5, 6], [7, 8, 5]), {}), (([1], [2]), dict(pools=(0,))), (([1], [2]), dict(pools=(A, A + 8))),
                                     (([1], [2]), dict(page_bytes=0)), (([1], [2]), dict(page_bytes=24)), (([1], [2]), dict(page_bytes=-16)), (([1], [2]), dict(n_pages=-1)),
                                     (([1], [2]), dict(ctx=None))], ids=str)
def test_copies_refuse(args, kw):
    with pytest.raises(ValueError):
        copy(*args, **kw)


@pytest.mark.parametrize("kw", [dict(ctx=None), dict(dtype=2), dict(dtype=-1), dict(M=-1), dict(M=2 ** 31), dict(N=0), dict(N=-5), dict(ld=99), dict(x=None), dict(u=None), dict(out=None),
                                dict(x=A + 2), dict(x=A + 1, dtype=0)], ids=str)
def test_sample_refuses(kw):
    with pytest.raises(ValueError):
        sample(**kw)


def test_sample_does_not_support():
    with pytest.raises(NotImplementedError):
        sample(N=2 ** 20 + 1, ld=2 ** 21)


def test_nothing_to_do_needs_nothing():
    attn(B=0, table=None, lens=None, starts=None, q=None, k=None, v=None, out=None)
    attn(T=0, q=None, out=None)
    rope(B=0, qkv=None)
    rope(T=0, qkv=None)
    copy([], [])
    copy([1], [2], pools=())
    sample(M=0, x=None, u=None, out=None)


@pytest.mark.parametrize("name", ["table", "lens", "starts"])
def test_index_arrays_that_are_not_aligned(name):
    for call in (attn, rope):
        with pytest.raises(ValueError, match="aligned"):
            call(**{name: A + 2})


@pytest.mark.parametrize("name", ["u", "t", "k", "p", "q", "out", "prob"])
def test_row_arrays_that_are_not_aligned(name):
    with pytest.raises(ValueError, match="aligned"):
        sample(**{name: A + 1})


@pytest.mark.parametrize("q", [A, A + 16, A + 2 * 12 * 128 * 2 - 16, A - 2 * 8 * 128 * 2 + 16])
def test_append_refuses_queries_over_its_input(q):
    with pytest.raises(ValueError, match="overlaps"):
        rope(q=q)
