"""Products of ragged row groups and their gradients (csrc/ct_grouped.hip) against plain 64-bit loops over the groups.

Tolerances: a sum of c products in 32 bits, in any order and with an error of at most one unit (2^-23) for each addition, is off by at most
(c + 4) 2^-23 sum |x| |w|; scale and shift add two roundings of the value; storing in 16 bits adds half a step of the type."""
import importlib

import numpy as np
import pytest

grouped = importlib.import_module("3deecelltracker_amd.grouped")
_lib = importlib.import_module("3deecelltracker_amd._lib")

TYPES = ("float32", "bfloat16", "float16")
UNIT = 2.0 ** -23


def _torch():
    import torch
    return torch


def _rand(shape, dtype, seed, scale=1.0):
    t = _torch()
    g = t.Generator(device="cuda").manual_seed(seed)
    return (t.randn(*shape, generator=g, device="cuda") * scale).to(getattr(t, dtype))


def _offsets(counts):
    return [0] + np.cumsum(counts).tolist()


def _step(t, dtype):
    return 0.0 if dtype == t.float32 else t.finfo(dtype).eps / 2


def _check(got, want, bound, dtype):
    """|got - want| <= bound + half a step of the stored type (and the smallest value it holds)"""
    t = _torch()
    got = got.double().cpu()
    tol = bound * (1 + 2.0 ** -8) + want.abs() * _step(t, dtype) + t.finfo(dtype).tiny
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} values off; worst {float(((got - want).abs() / tol).max())} of the tolerance at {tuple(int(v) for v in bad.nonzero()[0])}"


def _ref(x, w, counts, scale=None, shift=None, slope=1.0):
    t = _torch()
    x, w = x.double().cpu(), w.double().cpu()
    rows, k = x.shape
    y = t.zeros(rows, w.shape[2], dtype=t.float64); b = t.zeros_like(y)
    start = 0
    for g, c in enumerate(counts):
        xs = x[start:start + c]
        v, m = xs @ w[g], (k + 4) * UNIT * (xs.abs() @ w[g].abs())
        if scale is not None or shift is not None:
            sc = scale[g].double().cpu() if scale is not None else t.ones(w.shape[2], dtype=t.float64)
            sh = shift[g].double().cpu() if shift is not None else t.zeros(w.shape[2], dtype=t.float64)
            m = m * sc.abs() + 2 * UNIT * ((v * sc).abs() + sh.abs())
            v = v * sc + sh
        y[start:start + c] = t.where(v >= 0, v, v * slope)
        b[start:start + c] = m * max(1.0, abs(slope)) + UNIT * v.abs()
        start += c
    return y, b


CASES = [
    # counts of rows, K, N, rows behind the last group
    ([1], 1, 1, 0), ([1], 64, 64, 0), ([0, 1, 0], 61, 512, 0), ([5, 0, 0, 7], 3, 5, 2), ([64, 64], 64, 64, 0), ([65, 63, 1], 65, 129, 1),
    ([600, 613], 61, 512, 0), ([17], 512, 130, 3), ([0, 0, 0], 16, 16, 4), ([1] * 130, 48, 40, 0), ([3, 0] * 70, 33, 17, 9), ([300], 130, 1, 0),
    ([129, 2, 0, 258], 257, 255, 5), ([700, 1, 90], 128, 256, 0),
    # the large tiles: more of them than compute units, partial in every direction
    ([4000, 0, 3500, 777], 72, 2050, 3), ([2100, 1, 2300], 136, 1161, 0), ([0, 90, 64, 131, 77, 1, 200, 63, 65, 2], 1300, 1290, 1),
    ([33, 0, 100, 5] * 4, 520, 517, 2), ([9] * 20 + [0] * 10 + [31], 700, 264, 2), ([40, 31], 2050, 70, 0),
    # every rule by which a tile is chosen: runs of column tiles; deep and wide stages where tiles are few; both gradients in one launch
    ([9000, 12000, 11000], 72, 650, 5), ([1500, 1500], 320, 900, 0), ([62, 63] * 4, 300, 1500, 2), ([250] * 4, 200, 512, 0), ([1024, 1024], 512, 512, 0),
    ([4500, 4500], 40, 1000, 1), ([1] * 64, 200, 256, 0), ([300, 300], 515, 831, 0), ([3, 4] * 15, 333, 515, 0), ([250] * 14, 1300, 1290, 0), ([100] * 20, 300, 300, 3),
    # long sums for few columns, of even and odd width
    ([2, 0, 3], 3181, 16, 2), ([90, 1], 1024, 30, 0), ([100, 40], 1001, 333, 0), ([300, 41], 2755, 411, 1), ([33], 600, 1, 0),
    # long sums for few weights
    ([2300, 0, 1501], 61, 70, 3), ([1024, 1024], 61, 512, 0), ([5000], 128, 64, 1), ([1600, 3], 7, 33, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,k,n,tail", CASES, ids=lambda v: str(v)[:24])
def test_product(dtype, counts, k, n, tail):
    t = _torch()
    rows, g = sum(counts) + tail, len(counts)
    x, w = _rand((rows, k), dtype, 1), _rand((g, k, n), dtype, 2, k ** -0.5)
    if tail:
        x[-tail:] = float("nan")                                       # rows that belong to no group are not looked at
    y = grouped.product(x, w, _offsets(counts))
    want, bound = _ref(x.nan_to_num(0.0), w, counts)
    assert y.dtype == x.dtype and tuple(y.shape) == (rows, n)
    _check(y, want, bound, y.dtype)
    if tail:
        assert bool((y[-tail:] == 0).all())
    wide = grouped.product(x, w, _offsets(counts), out_dtype=t.float32)
    _check(wide, want, bound, t.float32)
    # a transposed view of weights laid out the other way, and the same said by the argument
    wt = w.transpose(1, 2).contiguous()
    for other in (grouped.product(x, wt.transpose(1, 2), _offsets(counts)), grouped.product(x, wt, _offsets(counts), transposed=True)):
        _check(other, want, bound, y.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts,k,n,tail", CASES, ids=lambda v: str(v)[:24])
def test_product_grad(dtype, counts, k, n, tail):
    t = _torch()
    rows, g = sum(counts) + tail, len(counts)
    x, w, dy = _rand((rows, k), dtype, 1), _rand((g, k, n), dtype, 2, k ** -0.5), _rand((rows, n), dtype, 3, 0.1)
    if tail:
        x[-tail:] = float("nan"); dy[-tail:] = float("inf")
    off = _offsets(counts)
    dx, dw = grouped.product_grad(dy, x, w, off)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and dx.shape == x.shape and dw.shape == w.shape
    clean = dy.clone()
    if tail:
        clean[-tail:] = 0
        assert bool((dx[-tail:] == 0).all())
    want, bound = _ref(clean, w.transpose(1, 2), counts)
    _check(dx, want, bound, dx.dtype)
    only_x = grouped.product_grad(dy, x, w, off, need_w=False)             # (alone it may take other tiles, so sum in another order)
    assert only_x[1] is None
    _check(only_x[0], want, bound, dx.dtype)
    xs, ds = x.double().cpu(), dy.double().cpu()
    want = t.stack([xs[a:b].T @ ds[a:b] for a, b in zip(off, off[1:])])
    bound = t.stack([(b - a + 4) * UNIT * (xs[a:b].abs().T @ ds[a:b].abs()) for a, b in zip(off, off[1:])])
    _check(dw, want, bound, dw.dtype)
    only_w = grouped.product_grad(dy, x, w, off, need_x=False, out_dtype=t.float32)
    assert only_w[0] is None
    _check(only_w[1], want, bound, t.float32)


@pytest.mark.gpu
def test_gradients_against_differences():
    """<dx, u> and <dw, v> equal the change of <y, dy> along u and v: y is linear in x and in w, so one difference is exact up to rounding"""
    t = _torch()
    counts, k, n = [20, 0, 33, 1], 37, 51
    x, w, dy = _rand((54, k), "float32", 1), _rand((4, k, n), "float32", 2), _rand((54, n), "float32", 3)
    u, v = _rand((54, k), "float32", 4), _rand((4, k, n), "float32", 5)
    off = _offsets(counts)
    dx, dw = grouped.product_grad(dy, x, w, off)
    f = lambda a, b: float((grouped.product(a, b, off).double() * dy.double()).sum())
    # each of the 54 n values of y is off by at most (k + 4) UNIT k max|x| max|w|, and so are the sums; 54 n |dy| of them
    tol = 54 * n * float(dy.abs().max()) * (k + 4) * UNIT * k * 40 * 2
    assert abs(f(u, w) - float((dx.double() * u.double()).sum())) <= tol
    assert abs(f(x, v) - float((dw.double() * v.double()).sum())) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("use", ["scale", "shift", "both", "one row"])
def test_normalisation_and_activation(dtype, use):
    t = _torch()
    counts, k, n = [40, 0, 71], 61, 131
    x, w = _rand((111, k), dtype, 1), _rand((3, k, n), dtype, 2, k ** -0.5)
    sc = _rand((3, n), "float32", 3) if use != "shift" else None
    sh = _rand((3, n), "float32", 4) if use != "scale" else None
    if use == "one row":
        sc, sh = sc[0], sh[1]
    y = grouped.product(x, w, _offsets(counts), scale=sc, shift=sh, slope=0.3)
    full = lambda a: None if a is None else a.expand(3, n)
    want, bound = _ref(x, w, counts, full(sc), full(sh), 0.3)
    _check(y, want, bound, y.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k,n,pad", [(61, 77, 3), (64, 128, 8), (64, 128, 1), (128, 256, 64)])
def test_rows_inside_wider_tensors(dtype, k, n, pad):
    """Operands that are slices of tensors full of NaN, a result inside a tensor that has to stay as it is"""
    t = _torch()
    counts = [70, 3, 0, 60]
    rows = sum(counts) + 6
    nan = float("nan")
    xb = t.full((rows + 2, k + pad), nan, device="cuda", dtype=getattr(t, dtype)); x = xb[1:-1, pad // 2:pad // 2 + k]
    wb = t.full((5, k + 2, n + pad), nan, device="cuda", dtype=getattr(t, dtype)); w = wb[1:, 1:-1, pad // 2:pad // 2 + n]
    db = t.full((rows + 2, n + pad), nan, device="cuda", dtype=getattr(t, dtype)); dy = db[1:-1, pad // 2:pad // 2 + n]
    x[:-6].copy_(_rand((rows - 6, k), dtype, 1)); w.copy_(_rand((4, k, n), dtype, 2, k ** -0.5)); dy[:-6].copy_(_rand((rows - 6, n), dtype, 3))
    yb = t.full((rows + 2, n + pad), 7.0, device="cuda", dtype=getattr(t, dtype)); y = yb[1:-1, pad // 2:pad // 2 + n]
    off = _offsets(counts)
    assert grouped.product(x, w, off, out=y) is y
    want, bound = _ref(x.nan_to_num(0.0), w, counts)
    _check(y[:-6], want[:-6], bound[:-6], y.dtype)
    assert bool((y[-6:] == 7).all())                                    # rows behind the last group stay as they were
    y[:-6] = 7.0
    assert bool((yb == 7).all())
    dx, dw = grouped.product_grad(dy, x, w, off)
    want, bound = _ref(dy.nan_to_num(0.0), w.transpose(1, 2), counts)
    _check(dx, want, bound, dx.dtype)
    dwc = grouped.product_grad(dy.contiguous(), x.contiguous(), w.contiguous(), off)[1]
    assert t.equal(dw, dwc) or bool(((dw.float() - dwc.float()).abs() <= 2.0 ** -7 * dwc.float().abs() + 1e-3).all())
    assert bool(t.isfinite(dw).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite_stay_in_their_rows(dtype):
    t = _torch()
    counts, k, n = [70, 66, 64], 96, 80
    x, w = _rand((200, k), dtype, 1), _rand((3, k, n), dtype, 2, k ** -0.5)
    clean = grouped.product(x, w, _offsets(counts))
    x[5, 7] = float("nan"); x[80, 95] = float("inf"); w[2, 3, 9] = float("nan")
    y = grouped.product(x, w, _offsets(counts))
    assert bool(t.isnan(y[5]).all()) and not bool(t.isfinite(y[80]).any()) and bool(t.isnan(y[136:, 9]).all())
    keep = t.ones_like(y, dtype=t.bool)
    keep[5] = keep[80] = False; keep[136:, 9] = False
    assert t.equal(y[keep], clean[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k,n", [(96, 80), (300, 260), (61, 40)])
def test_values_that_are_not_finite_stay_in_their_group(dtype, k, n):
    """A stage of the sum over a group's rows may begin in its neighbour's: what stands there does not count"""
    t = _torch()
    counts = [70, 1, 66, 0, 130, 7]
    x, dy, w = _rand((280, k), dtype, 1), _rand((280, n), dtype, 2), _rand((6, k, n), dtype, 3)
    off = _offsets(counts)
    clean = grouped.product_grad(dy, x, w, off)
    x[100, :] = float("nan"); dy[71:137] = float("inf"); x[274:] = float("nan"); dy[274:] = float("nan")       # group 2, and behind the last
    dx, dw = grouped.product_grad(dy, x, w, off)
    for g in (0, 1, 3, 4, 5):
        assert t.equal(dw[g], clean[1][g]), g
    assert not bool(t.isfinite(dw[2]).any()) and t.equal(dx[:71], clean[0][:71]) and t.equal(dx[137:274], clean[0][137:274])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_offsets_past_32_bits(dtype):
    """Rows and weight blocks whose first value lies more than 2^31 values into the tensor"""
    t = _torch()
    x = t.zeros(70000, 40000, device="cuda", dtype=getattr(t, dtype))[:, :64]
    w = t.zeros(3, 40000, 40000, device="cuda", dtype=getattr(t, dtype))[:, -64:, -96:] if dtype == "bfloat16" else _rand((3, 64, 96), dtype, 2)
    x[-80:].copy_(_rand((80, 64), dtype, 1)); w[1:].copy_(_rand((2, 64, 96), dtype, 3, 0.1))
    off = [0, 69000, 69930, 70000]
    y = grouped.product(x, w, off)
    want, bound = _ref(x[-80:], w[1:], [10, 70])
    _check(y[-80:], want, bound, y.dtype)
    dy = _rand((70000, 96), dtype, 4)
    dx, dw = grouped.product_grad(dy, x, w, off)
    want, bound = _ref(dy[-80:], w[1:].transpose(1, 2), [10, 70])
    _check(dx[-80:], want, bound, dx.dtype)
    xs, ds = x[-70:].double().cpu(), dy[-70:].double().cpu()
    _check(dw[2], xs.T @ ds, (74 * UNIT) * (xs.abs().T @ ds.abs()), dw.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_shared_block_equals_one_group(dtype):
    t = _torch()
    counts = [33, 0, 190, 64]
    x, w = _rand((287, 61), dtype, 1), _rand((1, 61, 96), dtype, 2, 0.1)
    a = grouped.product(x, w.expand(4, 61, 96), _offsets(counts))
    want, bound = _ref(x, w.expand(4, 61, 96), counts)
    _check(a, want, bound, a.dtype)


@pytest.mark.gpu
def test_offsets_on_the_device_and_streams_and_graphs():
    """Offsets that a router summed on the device; the same call on another stream, twice at once, captured and replayed with other rows"""
    t = _torch()
    counts = [100, 0, 31, 200, 1]
    x, w = _rand((340, 128), "bfloat16", 1), _rand((5, 128, 192), "bfloat16", 2, 0.1)
    dy = _rand((340, 192), "bfloat16", 3)
    dev_off = t.cat([t.zeros(1, device="cuda", dtype=t.int64), t.tensor(counts, device="cuda").cumsum(0)]).to(t.int32)
    y = grouped.product(x, w, _offsets(counts))
    dx, dw = grouped.product_grad(dy, x, w, dev_off)
    assert t.equal(grouped.product(x, w, dev_off), y)
    t.cuda.synchronize()
    s1, s2 = t.cuda.Stream(), t.cuda.Stream()
    with t.cuda.stream(s1):
        a = [grouped.product(x, w, dev_off) for _ in range(4)]
    with t.cuda.stream(s2):
        b = [grouped.product_grad(dy, x, w, dev_off) for _ in range(4)]
    t.cuda.synchronize()
    assert all(t.equal(v, y) for v in a) and all(t.equal(v, dx) and t.equal(u, dw) for v, u in b)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        with pytest.raises(ValueError):
            grouped.product(x, w, _offsets(counts))                      # numbers on the host cannot be uploaded here
        gy = grouped.product(x, w, dev_off); gx, gw = grouped.product_grad(dy, x, w, dev_off)
    for seed, c in ((11, counts), (12, [0, 0, 340, 0, 0]), (13, [68] * 5), (14, [1, 2, 3, 4, 5])):
        x.copy_(_rand((340, 128), "bfloat16", seed)); dev_off.copy_(t.tensor(_offsets(c), dtype=t.int32))
        graph.replay()
        t.cuda.synchronize()
        ey = grouped.product(x, w, dev_off); ex, ew = grouped.product_grad(dy, x, w, dev_off)
        assert t.equal(gy, ey) and t.equal(gx, ex) and t.equal(gw, ew)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_sums_in_parts_in_a_graph_with_other_groups(dtype):
    """Long sums for few weights: the parts of each group are counted on the device, whatever the offsets hold when the graph is replayed"""
    t = _torch()
    x, dy, w = _rand((4000, 61), dtype, 1), _rand((4000, 70), dtype, 2, 0.1), _rand((3, 61, 70), dtype, 3, 0.1)
    off = t.tensor([0, 2000, 2000, 4000], dtype=t.int32, device="cuda")
    grouped.product_grad(dy, x, w, off)
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        dx, dw = grouped.product_grad(dy, x, w, off, out_dtype=t.float32)
    xs, ds = x.double().cpu(), dy.double().cpu()
    for o in ([0, 2000, 2000, 4000], [0, 0, 0, 4000], [0, 1, 2, 3], [0, 4000, 4000, 4000], [0, 1333, 2666, 3999], [0, 0, 0, 0]):
        off.copy_(t.tensor(o, dtype=t.int32))
        graph.replay()
        t.cuda.synchronize()
        want = t.stack([xs[a:b].T @ ds[a:b] for a, b in zip(o, o[1:])])
        bound = t.stack([(b - a + 4) * UNIT * (xs[a:b].abs().T @ ds[a:b].abs()) for a, b in zip(o, o[1:])])
        _check(dw, want, bound, t.float32)
        ex, ew = grouped.product_grad(dy, x, w, off, out_dtype=t.float32)
        assert t.equal(dw, ew) and t.equal(dx, ex)
    for o in ([0, 3900, 10, 4000], [4000, 0, 4000, 0]):                  # not rising: any values, nothing outside
        off.copy_(t.tensor(o, dtype=t.int32))
        graph.replay()
        t.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_that_do_not_rise_stay_inside():
    """Numbers on the device are not looked at by the host: whatever they hold, nothing outside the result is written"""
    t = _torch()
    x, w = _rand((100, 64), "float16", 1), _rand((3, 64, 64), "float16", 2)
    box = t.full((120, 64), 5.0, device="cuda", dtype=t.float16)
    for off in ([0, 90, 10, 4000], [-7, 50, 20, 100], [0, -5, -9, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 0, 50]):
        d = t.tensor(off, dtype=t.int32, device="cuda")
        grouped.product(x, w, d, out=box[10:110])
        grouped.product_grad(x, x, w, d)
        t.cuda.synchronize()
        assert bool((box[:10] == 5).all()) and bool((box[110:] == 5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [64, 65, 1000, 20000])
def test_many_groups(groups):
    t = _torch()
    rng = np.random.default_rng(groups)
    counts = np.bincount(rng.integers(0, groups, 300), minlength=groups).tolist()
    x, w = _rand((300, 48), "bfloat16", 1), _rand((groups, 48, 32), "bfloat16", 2, 0.2)
    y = grouped.product(x, w, _offsets(counts))
    group = np.repeat(np.arange(groups), counts)
    xs, ws = x.double().cpu(), w.double().cpu()[group]
    _check(y, (xs[:, None] @ ws)[:, 0], (52 * UNIT) * (xs.abs()[:, None] @ ws.abs())[:, 0], y.dtype)
    dw = grouped.product_grad(y, x, w, _offsets(counts), need_x=False)[1]
    assert bool((dw[t.tensor(counts, device="cuda") == 0] == 0).all())
    one = int(np.argmax(counts)); a = _offsets(counts)[one]; b = a + counts[one]
    ys = y[a:b].double().cpu()
    _check(dw[one], xs[a:b].T @ ys, ((b - a + 4) * UNIT) * (xs[a:b].abs().T @ ys.abs()), dw.dtype)


@pytest.mark.gpu
def test_gradients_of_a_shared_block():
    t = _torch()
    counts, w = [50, 0, 70], _rand((1, 61, 40), "float32", 1)
    x, dy = _rand((120, 61), "float32", 2), _rand((120, 40), "float32", 3)
    dx, dw = grouped.product_grad(dy, x, w.expand(3, 61, 40), _offsets(counts))
    want, bound = _ref(dy, w.expand(3, 61, 40).transpose(1, 2), counts)
    _check(dx, want, bound, dx.dtype)
    whole = grouped.product_grad(dy, x, w, [0, 120])[1]
    xs, ds = x.double().cpu(), dy.double().cpu()
    _check(dw.sum(0, keepdim=True), (xs.T @ ds)[None], (2 * 124 * UNIT) * (xs.abs().T @ ds.abs())[None], t.float32)
    _check(whole, (xs.T @ ds)[None], (124 * UNIT) * (xs.abs().T @ ds.abs())[None], t.float32)


@pytest.mark.gpu
def test_empty_batch():
    t = _torch()
    x, w = t.empty(0, 61, device="cuda"), _rand((2, 61, 16), "float32", 1)
    assert tuple(grouped.product(x, w, [0, 0, 0]).shape) == (0, 16)
    dx, dw = grouped.product_grad(t.empty(0, 16, device="cuda"), x, w, [0, 0, 0])
    assert tuple(dx.shape) == (0, 61) and bool((dw == 0).all())


@pytest.mark.gpu
def test_refusals():
    t = _torch()
    x, w = _rand((10, 8), "float32", 1), _rand((2, 8, 6), "float32", 2)
    off = [0, 4, 10]
    dy = _rand((10, 6), "float32", 3)
    bad = [
        lambda: grouped.product(x.cpu(), w, off), lambda: grouped.product(x.double(), w.double(), off), lambda: grouped.product(x, w.half(), off),
        lambda: grouped.product(x, w[0], off), lambda: grouped.product(x[:, :7], w, off), lambda: grouped.product(x, w, [0, 10]),
        lambda: grouped.product(x, w, [0, 5, 11]), lambda: grouped.product(x, w, [0, 5, 4]), lambda: grouped.product(x, w, [1, 5, 10]),
        lambda: grouped.product(x, w, t.tensor(off, device="cuda")), lambda: grouped.product(x, w, t.tensor(off + [10], dtype=t.int32, device="cuda")),
        lambda: grouped.product(x.T.contiguous().T, w, off), lambda: grouped.product(x[:1].expand(10, 8), w, off),
        lambda: grouped.product(x, w, off, out=t.empty(10, 7, device="cuda")), lambda: grouped.product(x, w, off, out=t.empty(10, 6, device="cuda").half()),
        lambda: grouped.product(x, w, off, out=x[:, :6]), lambda: grouped.product(x, w, off, out_dtype=t.float16),
        lambda: grouped.product(x, w, off, scale=t.ones(5, device="cuda")), lambda: grouped.product(x, w, off, shift=t.ones(3, 6, device="cuda")),
        lambda: grouped.product(x, w, off, scale=t.ones(6)), lambda: grouped.product(x, w.clone().requires_grad_(), off),
        lambda: grouped.product(x, w[:, :, ::2], off), lambda: grouped.product(x[:, :0], w[:, :0], off),
        lambda: grouped.product_grad(dy[:9], x, w, off), lambda: grouped.product_grad(dy.half(), x, w, off),
        lambda: grouped.product_grad(dy, x, w, off, out_dtype=t.bfloat16),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


def test_the_abi_refuses_without_a_gpu():
    if not _lib.LIB_PATH.exists():
        importlib.import_module("__graft_entry__").build()
    L = _lib.lib()
    ok = dict(type=0, out=0, x=64, ldx=8, rows=4, K=8, w=64, wg=48, ldw=6, wt=0, N=6, off=64, G=2, sc=None, sh=None, ag=0, slope=1.0, fill=1, y=64, ldy=6,
              st=None)
    call = lambda **kw: L.ct_grouped_product(*{**ok, **kw}.values())
    for kw in (dict(type=3), dict(type=-1), dict(out=1), dict(rows=-1), dict(K=0), dict(N=0), dict(G=0), dict(x=None), dict(w=None), dict(off=None), dict(y=None),
               dict(ldx=7), dict(ldw=5), dict(ldy=5), dict(wg=-1), dict(ag=-1), dict(wt=1, ldw=7)):
        assert call(**kw) == _lib.CT_EINVAL, kw
    assert call(rows=0) == 0 and call(G=2 ** 16 + 1) == _lib.CT_ESHAPE
    assert call(rows=2 ** 31 - 1, N=2 ** 20, ldw=2 ** 20, ldy=2 ** 20) == _lib.CT_ESHAPE
    ok2 = dict(type=0, out=0, dy=64, lddy=6, x=64, ldx=8, rows=4, K=8, w=64, wg=48, ldw=6, wt=0, N=6, off=64, G=2, dx=64, lddx=8, dw=64, dwg=48, lddw=6, ws=None,
               wsb=0, st=None)
    call2 = lambda **kw: L.ct_grouped_product_grad(*{**ok2, **kw}.values())
    for kw in (dict(type=3), dict(out=2), dict(rows=-1), dict(K=0), dict(N=0), dict(G=0), dict(x=None), dict(dy=None), dict(w=None), dict(off=None), dict(ldx=7),
               dict(lddy=5), dict(ldw=5), dict(lddw=5), dict(dwg=47), dict(lddx=7), dict(wg=-1), dict(wt=1, ldw=7)):
        assert call2(**kw) == _lib.CT_EINVAL, kw
    assert L.ct_grouped_product_grad_workspace_bytes(0, 4, 8, 6, 2) == 0 and L.ct_grouped_product_grad_workspace_bytes(0, 2048, 8, 6, 2) > 0
    assert call2(rows=2048) == _lib.CT_EINVAL and call2(rows=2048, ws=64, wsb=8) == _lib.CT_EWORKSPACE
    for kw in (dict(ldx=2 ** 22 + 1), dict(lddy=2 ** 22 + 1), dict(ldw=2 ** 22 + 1)):
        assert call2(**kw) == _lib.CT_ESHAPE, kw
