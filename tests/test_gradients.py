"""The global gradient norm and clipping (csrc/ct_gradnorm.hip) against 64-bit sums.

Tolerances: squares are summed in 64 bits, so the norm is off by its one rounding to 32 bits (2^-24, and 2^-40 for the sum); a clipped value carries
the rounding of the factor and of the product to 32 bits (2^-24 each) and half a step of its type."""
import importlib
import math

import numpy as np
import pytest

gradients = importlib.import_module("3deecelltracker_amd.gradients")
_lib = importlib.import_module("3deecelltracker_amd._lib")

TYPES = ("float32", "bfloat16", "float16")
HALF = 2.0 ** -24


def _torch():
    import torch
    return torch


def _list(sizes, types, seed=0, scale=1.0):
    t = _torch()
    g = t.Generator(device="cuda").manual_seed(seed)
    return [(t.randn(s, generator=g, device="cuda") * scale).to(getattr(t, types[i % len(types)])) for i, s in enumerate(sizes)]


def _check(out, norm, grads, clip):
    t = _torch()
    want = math.sqrt(math.fsum(float((g.double() ** 2).sum()) for g in grads))
    assert norm.dtype == t.float32 and norm.dim() == 0
    if want > 2.0 ** 128 * (1 - 2.0 ** -25):                             # 5003 values around 1e37: 7.0e38, rounded to 32 bits that is infinity
        assert math.isinf(float(norm))
    else:
        assert abs(float(norm) - want) <= want * (HALF + 2.0 ** -40)
    f = clip / max(want, clip)
    for i, (o, g) in enumerate(zip(out, grads)):
        e = g.double() * f
        tol = e.abs() * (2 * HALF * (1 + 2.0 ** -10) + t.finfo(g.dtype).eps / 2 * (1 + 2.0 ** -10)) + t.finfo(g.dtype).smallest_normal * t.finfo(g.dtype).eps
        assert o.dtype == g.dtype and o.shape == g.shape and bool(((o.double() - e).abs() <= tol).all()), i


SIZES = [[1], [4096], [4097], [0, 5, 0], [3, 1, 2, 7, 15, 16, 17], [10000, 1, 0, 4096, 8193], [1] * 300, [65, 0] * 130 + [100003]]


@pytest.mark.gpu
@pytest.mark.parametrize("types", [("float32",), ("bfloat16",), ("float16",), TYPES], ids="-".join)
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: str(s)[:20])
def test_norm_and_clip(types, sizes):
    t = _torch()
    grads = _list(sizes, types)
    keep = [g.clone() for g in grads]
    for clip in (0.25, 1e9):
        out = [t.empty_like(g) for g in grads]
        s = gradients.GradientSet(grads, out=out)
        assert s.out[0] is out[0] and len(s.out) == len(grads)
        norm = s.clip(clip)
        _check(out, norm, keep, clip)
        assert t.equal(s.norm(), norm)
        assert all(t.equal(a, b) for a, b in zip(grads, keep))
        if clip == 1e9:
            assert all(t.equal(a, b) for a, b in zip(out, keep))
    got, norm = gradients.clip_by_global_norm(grads, 0.25)              # in place
    assert all(a is b for a, b in zip(got, grads))
    _check(grads, norm, keep, 0.25)
    got, norm = gradients.clip_by_global_norm(keep, 0.25, out=[t.empty_like(g) for g in keep])
    assert all(t.equal(a, b) for a, b in zip(got, grads))


@pytest.mark.gpu
def test_large_tensors_repeat_bit_for_bit():
    t = _torch()
    grads = _list([12_000_001, 3, 5_000_000], ("bfloat16", "float32"), seed=3, scale=0.01)
    s = gradients.GradientSet(grads, out=[t.empty_like(g) for g in grads])
    a = s.clip(0.5)
    first = [o.clone() for o in s.out]
    _check(s.out, a, grads, 0.5)
    for _ in range(3):
        assert t.equal(s.clip(0.5), a) and all(t.equal(x, y) for x, y in zip(first, s.out))


@pytest.mark.gpu
def test_a_tensor_past_32_bits():
    t = _torch()
    g = t.zeros(2 ** 31 + 4101, dtype=t.bfloat16, device="cuda")
    g[-3:] = t.tensor([3.0, -4.0, 12.0], device="cuda"); g[1] = 84.0
    out, norm = gradients.clip_by_global_norm([g], 8.5)
    assert float(norm) == 85.0 and out[0][-3:].tolist() == [0.30078125, -0.400390625, 1.203125] and float(out[0][1]) == 8.375   # a tenth, rounded to bf16
    assert int(t.count_nonzero(out[0])) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5, 8])
def test_slices_of_one_buffer(offset):
    """Gradients end to end in a bucket: any alignment of a value; what lies between them stays as it was"""
    t = _torch()
    for dtype in TYPES:
        buf = t.full((60000,), 9.0, device="cuda", dtype=getattr(t, dtype))
        sizes, views, at = [1, 4099, 17, 0, 20001], [], offset
        for n in sizes:
            views.append(buf[at:at + n]); at += n + 1
        for v, g in zip(views, _list(sizes, (dtype,), seed=offset)):
            v.copy_(g)
        keep = [v.clone() for v in views]
        norm = gradients.GradientSet(views).clip(0.5)
        _check(views, norm, keep, 0.5)
        for v in views:
            v.fill_(9.0)
        assert bool((buf == 9).all())


@pytest.mark.gpu
def test_tensors_in_another_order_of_indices():
    t = _torch()
    a = _list([6 * 50 * 70], ("float32",))[0].view(6, 50, 70)
    grads = [a.permute(2, 0, 1), _list([5], ("float16",))[0].view(1, 5, 1)]
    keep = [g.clone() for g in grads]
    norm = gradients.GradientSet(grads).clip(1.0)
    _check(grads, norm, keep, 1.0)


@pytest.mark.gpu
def test_extreme_values():
    t = _torch()
    for scale in (1e-30, 1e30, 1e37):                                    # squares beyond the 32-bit range on either side
        grads = _list([5000, 3], ("float32", "bfloat16"), scale=scale)
        keep = [g.clone() for g in grads]
        _check(*gradients.clip_by_global_norm(grads, 1.0), keep, 1.0)
    big = [t.full((64,), 3e38, device="cuda")]                            # the norm itself is beyond 32 bits: reported as infinity, the gradients are fine
    out, norm = gradients.clip_by_global_norm(big, 2.0)
    assert math.isinf(float(norm)) and bool(((out[0] - 0.25).abs() <= 1e-6).all())
    for value in (float("nan"), float("inf"), -float("inf")):
        grads = _list([5000, 0, 77], TYPES)
        grads[2][5] = value
        out, norm = gradients.clip_by_global_norm(grads, 1.0)
        assert not math.isfinite(float(norm)) and all(bool(t.isnan(o).all()) for o in out)
    zero = [t.zeros(100, device="cuda")]
    out, norm = gradients.clip_by_global_norm(zero, 1.0)
    assert float(norm) == 0 and bool((out[0] == 0).all())
    assert float(gradients.GradientSet([]).norm()) == 0.0 and gradients.clip_by_global_norm([], 1.0)[0] == []


@pytest.mark.gpu
def test_streams_and_graphs():
    t = _torch()
    grads = _list([40000, 3, 513], TYPES)
    s = gradients.GradientSet(grads, out=[t.empty_like(g) for g in grads])
    want = s.norm()
    t.cuda.synchronize()
    streams = [t.cuda.Stream() for _ in range(3)]
    norms = []
    for st in streams:
        with t.cuda.stream(st):
            norms += [s.norm() for _ in range(5)]
    t.cuda.synchronize()
    assert all(t.equal(n, want) for n in norms)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        n1 = s.clip(0.5)
        out2, n2 = gradients.clip_by_global_norm(grads, 0.5, out=[t.empty_like(g) for g in grads])
        with pytest.raises(ValueError):
            gradients.GradientSet(grads)
    for seed in range(1, 5):
        for g, v in zip(grads, _list([40000, 3, 513], TYPES, seed=seed)):
            g.copy_(v)
        graph.replay()
        t.cuda.synchronize()
        _check(s.out, n1, grads, 0.5); _check(out2, n2, grads, 0.5)


@pytest.mark.gpu
def test_refusals():
    t = _torch()
    a, b = t.ones(100, device="cuda"), t.ones(100, device="cuda")
    bad = [
        lambda: gradients.GradientSet([a.cpu()]), lambda: gradients.GradientSet([a.double()]), lambda: gradients.GradientSet([a[::2]]),
        lambda: gradients.GradientSet([a[:1].expand(5)]), lambda: gradients.GradientSet([a, a]), lambda: gradients.GradientSet([a[:60], a[50:]]),
        lambda: gradients.GradientSet([a], out=[b, b]), lambda: gradients.GradientSet([a], out=[b.half()]), lambda: gradients.GradientSet([a], out=[b[:99]]),
        lambda: gradients.GradientSet([a, b], out=[b, t.empty_like(a)]), lambda: gradients.GradientSet([a[:50], b], out=[a[10:60], b]),
        lambda: gradients.GradientSet([a.view(10, 10)], out=[b.view(10, 10).T]), lambda: gradients.GradientSet([3.0]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    s = gradients.GradientSet([a])
    for clip in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            s.clip(clip)
    assert float(gradients.GradientSet([a, a], out=[b, t.empty_like(a)]).norm()) == pytest.approx(math.sqrt(200))   # read twice, written apart


def test_the_abi_refuses_without_a_gpu():
    import ctypes as C
    if not _lib.LIB_PATH.exists():
        importlib.import_module("__graft_entry__").build()
    L = _lib.lib()
    sizes, types = (C.c_int64 * 2)(5, 4097), (C.c_int * 2)(0, 1)
    ptr = (C.c_void_p * 2)(64, 128)
    assert L.ct_gradset_chunks(2, sizes) == 3 and L.ct_gradset_chunks(0, None) == 0 and L.ct_gradset_chunks(1, (C.c_int64 * 1)(-1)) == -1
    need = L.ct_gradset_table_bytes(2)
    write = lambda n=2, i=ptr, o=ptr, s=sizes, ty=types, table=64, nb=need: L.ct_gradset_write(n, i, o, s, ty, table, nb, None)
    for kw in (dict(n=-1), dict(i=None), dict(s=None), dict(ty=None), dict(table=None), dict(table=4), dict(s=(C.c_int64 * 2)(5, -1)), dict(ty=(C.c_int * 2)(0, 3)),
               dict(i=(C.c_void_p * 2)(64, None)), dict(o=(C.c_void_p * 2)(64, 129)), dict(i=(C.c_void_p * 2)(66, 128))):
        assert write(**kw) == _lib.CT_EINVAL, kw
    assert write(nb=need - 1) == _lib.CT_EWORKSPACE
    wb = L.ct_gradset_workspace_bytes()
    clip = lambda table=64, n=2, ch=3, c=1.0, norm=64, ws=64, nb=wb: L.ct_gradset_clip(table, n, ch, c, norm, ws, nb, None)
    for kw in (dict(table=None), dict(n=-1), dict(ch=-1), dict(c=0.0), dict(c=-1.0), dict(c=float("nan")), dict(c=float("inf")), dict(norm=None), dict(ws=None), dict(ws=4)):
        assert clip(**kw) == _lib.CT_EINVAL, kw
    assert clip(nb=wb - 1) == _lib.CT_EWORKSPACE and L.ct_gradset_norm(64, 2, 3, 64, 64, wb - 1, None) == _lib.CT_EWORKSPACE
