"""Gradients of the grouped products against differences and 64-bit sums, with bounds that come from the data: a sum of c products is off by at most
(c + 4) 2^-23 of the sum of their absolute values."""
import importlib

import pytest

grouped = importlib.import_module("3deecelltracker_amd.grouped")
from test_grouped import TYPES, UNIT, _check, _offsets, _rand


def _dx64(dy, w, off):
    import torch as t
    return t.cat([dy[a:b].double() @ w[g].double().T.contiguous() for g, (a, b) in enumerate(zip(off, off[1:]))])


def _dw64(x, dy, off):
    import torch as t
    return t.stack([x[a:b].double().T.contiguous() @ dy[a:b].double() for a, b in zip(off, off[1:])])


@pytest.mark.gpu
@pytest.mark.parametrize("counts,k,n", [([20, 0, 33, 1], 37, 51), ([300, 260], 512, 512), ([90], 61, 1), ([5] * 40, 300, 128)], ids=lambda v: str(v)[:20])
def test_gradients_against_differences(counts, k, n):
    """y is linear in x and in w, so <y, dy> changes by exactly <dx, u> along u and by <dw, v> along v.  u and v point along the gradients: what is
    compared is their squared norm, and a gradient that is scaled by 1.01, or zero, is off by more than the bound."""
    import torch as t
    off, rows, groups = _offsets(counts), sum(counts), len(counts)
    x, w, dy = _rand((rows, k), "float32", 1), _rand((groups, k, n), "float32", 2), _rand((rows, n), "float32", 3)
    u, v = _dx64(dy, w, off).float(), _dw64(x, dy, off).float()
    dx, dw = grouped.product_grad(dy, x, w, off)
    f = lambda a, b: float((grouped.product(a, b, off).double() * dy.double()).sum())
    for change, gradient, direction, terms in ((f(u, w), dx, u, (_dx64(dy.abs(), w.abs(), off) * u.abs().double()).sum()),
                                               (f(x, v), dw, v, (_dw64(x.abs(), dy.abs(), off) * v.abs().double()).sum())):
        # both sides are sums of the same products x w dy: of k (and rows for dw, n for dx) at a time in 32 bits, the rest in 64
        tol = (k + max(n, rows) + 8) * UNIT * float(terms)
        inner = lambda g: float((g.double() * direction.double()).sum())
        assert abs(change - inner(gradient)) <= tol
        assert abs(change - 1.01 * inner(gradient)) > tol and abs(change) > tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k,n,pad", [(61, 77, 3), (64, 128, 8), (64, 128, 1), (128, 256, 64), (200, 300, 5)])
@pytest.mark.parametrize("odd", ["x", "dy", "both"])
def test_dw_of_rows_inside_wider_tensors(dtype, k, n, pad, odd):
    """One operand or both a slice of a tensor full of NaN, rows of any stride and alignment"""
    import torch as t
    counts = [70, 3, 0, 60, 131]
    off, rows = _offsets(counts), 264

    def inside(a):
        buf = t.full((rows + 2, a.shape[1] + pad), float("nan"), device="cuda", dtype=a.dtype)
        part = buf[1:-1, pad // 2:pad // 2 + a.shape[1]]
        part.copy_(a)
        return part
    x, dy, w = _rand((rows, k), dtype, 1), _rand((rows, n), dtype, 3), _rand((5, k, n), dtype, 2, k ** -0.5)
    xs, ds = (inside(x) if odd != "dy" else x), (inside(dy) if odd != "x" else dy)
    want = _dw64(x, dy, off).cpu()
    bound = t.stack([(b - a + 4) * UNIT * (x[a:b].double().abs().T.contiguous() @ dy[a:b].double().abs()) for a, b in zip(off, off[1:])]).cpu()
    dx, dw = grouped.product_grad(ds, xs, w, off)
    _check(dw, want, bound, dw.dtype)
    _check(grouped.product_grad(ds, xs, w, off, need_x=False, out_dtype=t.float32)[1], want, bound, t.float32)
    _check(dx, _dx64(dy, w, off).cpu(), (n + 4) * UNIT * _dx64(dy.abs(), w.abs(), off).cpu(), dx.dtype)
