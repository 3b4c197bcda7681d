"""Dense layers whose rows come in ragged groups, each group with its own weight block (csrc/ct_grouped.hip).

    product(x, w, offsets)           rows offsets[g] .. offsets[g + 1] of x times w[g], normalisation and LeakyReLU in the same pass
    product_grad(dy, x, w, offsets)  its gradients with respect to x and w

The FFN's second layer is such a product with two groups -- the reference cells with the upper half of its weights, the target cells
with the lower half (reference ffn.py:258-265) -- and FFN.train_on_batch is built on them; a bank of networks (one for each
recording, or experts that a router has chosen rows for) is the general case.

Tensors are torch tensors on the GPU: float32, bfloat16 or float16, rows of any stride, contiguous along the last index.  Everything is
enqueued on the current stream of the tensors' device and does not wait for it."""
from __future__ import annotations

from typing import Sequence, Union

from . import _dev, _lib

MAX_SIZE = (1 << 31) - 1      # rows, columns: the library's sizes have 32 bits, offsets too
MAX_GROUPS = 1 << 16          # every workgroup looks its group up among them, 64 at a time
_ready = None


def _env():
    """(torch, {type: CT_F32 / CT_BF16 / CT_F16}, the library), looked up once.  The kernels of a small layer take less time than a dozen look-ups: the
    calls below test everything they ask of their operands in one expression, and only where that fails find out what is wrong."""
    global _ready
    if _ready is None:
        t = _lib.require_gpu()
        _ready = (t, {t.float32: 0, t.bfloat16: 1, t.float16: 2}, _lib.lib())
    return _ready


def _check_tensor(t, types, name, a, dims, dtype, device):
    """What every operand has to be; dtype, device None: the first one"""
    if not isinstance(a, t.Tensor) or not a.is_cuda:
        raise ValueError(f"{name}: expected a tensor on the GPU")
    if a.dim() != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got the shape {tuple(a.shape)}")
    if a.dtype is not dtype:
        if dtype is not None:
            raise ValueError(f"{name}: values are {a.dtype}, expected {dtype}")
        if a.dtype not in types:
            raise ValueError(f"{name}: values of type {a.dtype} are not supported (float32, bfloat16, float16)")
    if device is not None and a.device != device:
        raise ValueError(f"{name}: is on {a.device}, the other tensors are on {device}")
    _no_grad(t, name, a, ", but this product is not part of torch's graph: pass {name}.detach() and use product_grad")


def _no_grad(t, name, a, instead):
    if a.requires_grad and t.is_grad_enabled():
        raise ValueError(f"{name}: requires grad{instead.format(name=name)}")


def _row_stride(name, rows, cols, row_stride, col_stride):
    """Stride of the rows of [rows, columns]; a single row or column may carry any stride."""
    if cols > 1 and col_stride != 1:
        raise ValueError(f"{name}: the last index must be contiguous, its stride is {col_stride}")
    if rows <= 1 or cols == 0:
        return cols or 1
    if row_stride < cols:
        raise ValueError(f"{name}: rows overlap (stride {row_stride} for {cols} columns)")
    return row_stride


def _capturing(t, device):
    """Whether the current stream of `device` is being captured into a graph"""
    if t._C._cuda_getDevice() == device.index:
        return t._C._cuda_isCurrentStreamCapturing()
    with t.cuda.device(device):
        return t._C._cuda_isCurrentStreamCapturing()


def offsets_device(offsets: Union[Sequence[int], "torch.Tensor"], groups: int, rows: int, device):
    """int32 [groups + 1] on `device`.  Numbers on the host (a sequence, an array, a CPU tensor) are checked and uploaded; a tensor that is on
    the device already (a router's counts, summed there) is taken as it is, since looking at it would wait for the stream."""
    t = _env()[0]
    if isinstance(offsets, t.Tensor) and offsets.is_cuda:
        if offsets.device == device and offsets.dtype is t.int32 and offsets.shape == (groups + 1,) and offsets.is_contiguous():
            return offsets
        if offsets.dtype is not t.int32 or offsets.dim() != 1 or offsets.shape[0] != groups + 1 or not offsets.is_contiguous():
            raise ValueError(f"offsets: expected a contiguous int32 tensor of {groups + 1} numbers, got {offsets.dtype} {tuple(offsets.shape)}")
        raise ValueError(f"offsets: are on {offsets.device}, the other tensors are on {device}")
    given = offsets.tolist() if hasattr(offsets, "tolist") else list(offsets)
    try:
        host = [int(v) for v in given]
    except (TypeError, ValueError, OverflowError):
        host = None
    if host is None or host != given:
        raise ValueError("offsets: must be whole numbers")
    if len(host) != groups + 1:
        raise ValueError(f"offsets: expected {groups + 1} numbers for {groups} groups, got {len(host)}")
    if host[0] != 0 or any(a > b for a, b in zip(host, host[1:])) or host[-1] > rows:
        raise ValueError(f"offsets: must rise from 0 to at most {rows} rows")
    if _capturing(t, device):
        raise ValueError("offsets: numbers on the host cannot be uploaded while a graph is captured; pass an int32 tensor on the device")
    return t.tensor(host, dtype=t.int32, pin_memory=True).to(device, non_blocking=True)      # (from pageable memory the copy would wait for the stream)


def _as_is(t, a, groups, n, device):
    return a is None or (isinstance(a, t.Tensor) and a.shape == (groups, n) and a.dtype is t.float32 and a.device == device and a.is_contiguous() and
                         not a.requires_grad)


def _affine(name, a, groups, n, device):
    """[n] or [groups, n] -> (tensor with contiguous rows, stride of its groups)"""
    t = _env()[0]
    if not isinstance(a, t.Tensor) or not a.is_cuda or a.device != device or a.dtype is not t.float32 or a.dim() not in (1, 2):
        raise ValueError(f"{name}: expected a float32 tensor [{n}] or [{groups}, {n}] on {device}")
    if a.shape[-1] != n or (a.dim() == 2 and a.shape[0] not in (1, groups)):
        raise ValueError(f"{name}: shape {tuple(a.shape)} does not fit {groups} groups of {n} columns")
    _no_grad(t, name, a, ", but the product has no gradient for it: apply a {name} that is learned outside, or pass {name}.detach()")
    a = a.contiguous()
    return a, n if a.dim() == 2 and a.shape[0] == groups and groups > 1 else 0


def _weights(name, w, transposed):
    """w [G][K][N] ([G][N][K] if transposed) -> (G, K, N, read transposed, row stride, group stride); a block may be laid out either way"""
    g, k, n = w.shape
    sg, sk, sn = w.stride()
    if transposed:
        k, n, sk, sn = n, k, sn, sk
    if g < 1 or g > MAX_GROUPS or n < 1 or k < 1:
        raise ValueError(f"{name}: shape {tuple(w.shape)} is empty or has more than {MAX_GROUPS} groups")
    flip = (sn != 1 and sk == 1 and n > 1) or (transposed and sk == 1 and not (sn == 1 and k > 1))
    ld = _row_stride(name, n, k, sn, sk) if flip else _row_stride(name, k, n, sk, sn)
    return g, k, n, flip, ld, 0 if g == 1 else sg


def _span(a):
    """The bytes from a tensor's first value to its last"""
    p = a.data_ptr()
    return p, p + (sum((s - 1) * st for s, st in zip(a.shape, a.stride())) + 1) * a.element_size() if a.numel() else p


def _overlap(a, b):
    (p, q), (r, s) = _span(a), _span(b)
    return p < s and r < q


def _on_device(t, device, call, *args):
    """call(*args, stream) with `device` current: entry points without a handle run on the calling thread's current device"""
    if t._C._cuda_getDevice() == device.index:
        return call(*args, t._C._cuda_getCurrentRawStream(device.index))
    with t.cuda.device(device):
        return call(*args, t._C._cuda_getCurrentRawStream(device.index))


def product(x, w, offsets, *, transposed: bool = False, scale=None, shift=None, slope: float = 1.0, out=None, out_dtype=None):
    """y[r] = act(scale[g] * (x[r] . w[g]) + shift[g]) for the rows offsets[g] <= r < offsets[g + 1]; act(v) = v or slope * v where v < 0.

    x [rows, K]; w [G, K, N] of the same type (transposed=True: [G, N, K]; w.expand(G, K, N) shares one block); offsets: G + 1 numbers, on
    the host or as int32 on the device; scale, shift: float32 [N] or [G, N].  Sums are held in 32 bits and rounded once to `out_dtype`
    (x's type, or float32).  Rows behind offsets[G] are zero in a new result and stay as they were in a given `out` [rows, N].  -> [rows, N]"""
    t, types, L = _env()
    xt, device = getattr(x, "dtype", None), getattr(x, "device", None)
    if not (xt in types and isinstance(w, t.Tensor) and w.dtype is xt and w.device == device and x.is_cuda and x.dim() == 2 and w.dim() == 3 and
            not x.requires_grad and not w.requires_grad):
        _check_tensor(t, types, "x", x, 2, None, None)
        _check_tensor(t, types, "w", w, 3, xt, device)
    rows, k = x.shape
    g, wk, n, flip, ldw, group_stride = _weights("w", w, transposed)
    if rows > MAX_SIZE or k > MAX_SIZE or n > MAX_SIZE:
        raise ValueError(f"x {tuple(x.shape)}, w {tuple(w.shape)}: sizes above {MAX_SIZE} are not supported")
    if wk != k:
        raise ValueError(f"x has {k} columns, the weight blocks have {wk} rows")
    ldx = _row_stride("x", rows, k, *x.stride())
    dtype = out_dtype or (xt if out is None else out.dtype)
    if dtype is not xt and dtype is not t.float32:
        raise ValueError(f"out_dtype: {dtype} is neither {xt} nor float32")
    off = offsets_device(offsets, g, rows, device)
    sc = sh = None
    stride = 0
    if scale is None and shift is None:
        pass
    elif _as_is(t, scale, g, n, device) and _as_is(t, shift, g, n, device):
        sc, sh, stride = scale, shift, n
    else:
        (sc, s1), (sh, s2) = ((None, None) if a is None else _affine(name, a, g, n, device) for name, a in (("scale", scale), ("shift", shift)))
        if s1 is not None and s2 is not None and s1 != s2:            # one for all groups, the other for each
            sc, sh, s1 = sc.expand(g, n).contiguous(), sh.expand(g, n).contiguous(), n
        stride = s1 if s1 is not None else s2
    fill = out is None
    if fill:
        out, ldy = t.empty((rows, n), dtype=dtype, device=device), n
    else:
        _check_tensor(t, types, "out", out, 2, dtype, device)
        if tuple(out.shape) != (rows, n):
            raise ValueError(f"out: shape {tuple(out.shape)}, expected {(rows, n)}")
        ldy = _row_stride("out", rows, n, *out.stride())
        for name, a in (("x", x), ("w", w), ("the offsets", off), ("scale", sc), ("shift", sh)):
            if a is not None and _overlap(out, a):
                raise ValueError(f"out: overlaps {name}")
    rc = _on_device(t, device, L.ct_grouped_product, types[xt], types[dtype], x.data_ptr(), ldx, rows, k, w.data_ptr(), group_stride, ldw, flip, n,
                    off.data_ptr(), g, sc if sc is None else sc.data_ptr(), sh if sh is None else sh.data_ptr(), stride, slope, fill, out.data_ptr(), ldy)
    if rc:
        _lib.check(rc, "ct_grouped_product")
    if not fill:
        t.autograd.graph.increment_version(out)               # (a graph that saved `out` learns that it holds other values now)
    return out


def product_grad(dy, x, w, offsets, *, need_x: bool = True, need_w: bool = True, out_dtype=None):
    """The gradients of product(x, w, offsets) (no scale, shift or slope) for dy [rows, N] -> (dx [rows, K] of x's type, dw [G, K, N] of
    `out_dtype`: w's type, or float32); None in the place of one that is not needed.  Rows behind offsets[G] get a zero dx, a group without
    rows a zero dw[g].  Of a block that w.expand shares, each group's part comes separately: sum them."""
    t, types, L = _env()
    xt, device = getattr(x, "dtype", None), getattr(x, "device", None)
    if not (xt in types and isinstance(w, t.Tensor) and isinstance(dy, t.Tensor) and w.dtype is xt and dy.dtype is xt and w.device == device and
            dy.device == device and x.is_cuda and x.dim() == 2 and w.dim() == 3 and dy.dim() == 2 and
            not x.requires_grad and not w.requires_grad and not dy.requires_grad):
        _check_tensor(t, types, "x", x, 2, None, None)
        _check_tensor(t, types, "w", w, 3, xt, device)
        _check_tensor(t, types, "dy", dy, 2, xt, device)
    rows, k = x.shape
    g, wk, n, flip, ldw, group_stride = _weights("w", w, False)
    if rows > MAX_SIZE or k > MAX_SIZE or n > MAX_SIZE:
        raise ValueError(f"x {tuple(x.shape)}, w {tuple(w.shape)}: sizes above {MAX_SIZE} are not supported")
    if wk != k or dy.shape != (rows, n):
        raise ValueError(f"dy {tuple(dy.shape)}, x {tuple(x.shape)} and w {tuple(w.shape)} do not fit each other")
    ldx, lddy = _row_stride("x", rows, k, *x.stride()), _row_stride("dy", rows, n, *dy.stride())
    dtype = out_dtype or xt
    if dtype is not xt and dtype is not t.float32:
        raise ValueError(f"out_dtype: {dtype} is neither {xt} nor float32")
    off = offsets_device(offsets, g, rows, device)
    dx = t.empty((rows, k), dtype=xt, device=device) if need_x else None
    dw, ws, need = None, None, 0
    if need_w:
        dw = t.empty((g, k, n), dtype=dtype, device=device)
        need = L.ct_grouped_product_grad_workspace_bytes(types[xt], rows, k, n, g)
        if need:
            ws = _dev.workspace(need, device)
    rc = _on_device(t, device, L.ct_grouped_product_grad, types[xt], types[dtype], dy.data_ptr(), lddy, x.data_ptr(), ldx, rows, k, w.data_ptr(),
                    group_stride, ldw, flip, n, off.data_ptr(), g, dx.data_ptr() if need_x else None, k, dw.data_ptr() if need_w else None, k * n, n,
                    ws.data_ptr() if need else None, need)
    if rc:
        _lib.check(rc, "ct_grouped_product_grad")
    return dx, dw
