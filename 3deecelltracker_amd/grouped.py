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

MAX_GROUPS = 1 << 20


def _types():
    t = _lib.require_gpu()
    return {t.float32: 0, t.bfloat16: 1, t.float16: 2}          # CT_F32, CT_BF16, CT_F16


def _check_matrix(name, a, dims, dtype=None, device=None):
    t = _lib.require_gpu()
    if not isinstance(a, t.Tensor) or not a.is_cuda:
        raise ValueError(f"{name}: expected a tensor on the GPU")
    if a.dim() != dims:
        raise ValueError(f"{name}: expected {dims} dimensions, got the shape {tuple(a.shape)}")
    if a.dtype not in _types():
        raise ValueError(f"{name}: values of type {a.dtype} are not supported (float32, bfloat16, float16)")
    if dtype is not None and a.dtype != dtype:
        raise ValueError(f"{name}: values are {a.dtype}, expected {dtype}")
    if device is not None and a.device != device:
        raise ValueError(f"{name}: is on {a.device}, the other tensors are on {device}")
    if a.requires_grad and t.is_grad_enabled():
        raise ValueError(f"{name}: requires grad, but this product is not part of torch's graph: pass {name}.detach() and use product_grad")


def _row_stride(name, a):
    """Stride of the rows of [..., rows, columns]; a single row or column may carry any stride."""
    rows, cols = a.shape[-2], a.shape[-1]
    if cols > 1 and a.stride(-1) != 1:
        raise ValueError(f"{name}: the last index must be contiguous (strides {tuple(a.stride())})")
    if rows <= 1 or cols == 0:
        return max(cols, 1)
    if a.stride(-2) < cols:
        raise ValueError(f"{name}: rows overlap (strides {tuple(a.stride())})")
    return a.stride(-2)


def offsets_device(offsets: Union[Sequence[int], "torch.Tensor"], groups: int, rows: int, device):
    """int32 [groups + 1] on `device`.  Numbers on the host (a sequence, an array, a CPU tensor) are checked and uploaded; a tensor that is on
    the device already (a router's counts, summed there) is taken as it is, since looking at it would wait for the stream."""
    t = _lib.require_gpu()
    if isinstance(offsets, t.Tensor) and offsets.is_cuda:
        if offsets.dtype != t.int32 or offsets.dim() != 1 or offsets.shape[0] != groups + 1 or not offsets.is_contiguous():
            raise ValueError(f"offsets: expected a contiguous int32 tensor of {groups + 1} numbers, got {offsets.dtype} {tuple(offsets.shape)}")
        if offsets.device != device:
            raise ValueError(f"offsets: are on {offsets.device}, the other tensors are on {device}")
        return offsets
    host = [int(v) for v in (offsets.tolist() if hasattr(offsets, "tolist") else offsets)]
    if len(host) != groups + 1:
        raise ValueError(f"offsets: expected {groups + 1} numbers for {groups} groups, got {len(host)}")
    if host[0] != 0 or any(a > b for a, b in zip(host, host[1:])) or host[-1] > rows:
        raise ValueError(f"offsets: must rise from 0 to at most {rows} rows")
    return t.tensor(host, dtype=t.int32).to(device)


def _affine(name, a, groups, n, device):
    t = _lib.require_gpu()
    if a is None:
        return None
    if not isinstance(a, t.Tensor) or not a.is_cuda or a.device != device or a.dtype != t.float32 or a.dim() not in (1, 2):
        raise ValueError(f"{name}: expected a float32 tensor [{n}] or [{groups}, {n}] on {device}")
    a = a.unsqueeze(0) if a.dim() == 1 else a
    if a.shape[1] != n or a.shape[0] not in (1, groups):
        raise ValueError(f"{name}: shape {tuple(a.shape)} does not fit {groups} groups of {n} columns")
    return a.expand(groups, n)


def _groups(w):
    """(transposed, row stride, group stride) of w [G][K][N]; a view with K contiguous is read transposed."""
    g, k, n = w.shape
    flip = n > 1 and w.stride(2) != 1 and k >= 1 and w.stride(1) == 1
    ld = _row_stride("w", w.transpose(1, 2) if flip else w)
    group = 0 if g == 1 else w.stride(0)
    if group < 0:
        raise ValueError("w: negative strides")
    return flip, ld, group


def _overlap(a, b):
    """Whether the byte ranges that two tensors span meet."""
    def span(x):
        last = sum((s - 1) * st for s, st in zip(x.shape, x.stride()))
        return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()
    if a.numel() == 0 or b.numel() == 0:
        return False
    (p, q), (r, s) = span(a), span(b)
    return p < s and r < q


def product(x, w, offsets, *, transposed: bool = False, scale=None, shift=None, slope: float = 1.0, out=None, out_dtype=None):
    """y[r] = act(scale[g] * (x[r] . w[g]) + shift[g]) for the rows offsets[g] <= r < offsets[g + 1]; act(v) = v or slope * v where v < 0.

    x [rows, K]; w [G, K, N] of the same type (transposed=True: [G, N, K]; w.expand(G, K, N) shares one block); offsets: G + 1 numbers, on
    the host or as int32 on the device; scale, shift: float32 [N] or [G, N].  Sums are held in 32 bits and rounded once to `out_dtype`
    (x's type, or float32).  Rows behind offsets[G] are zero in a new result and stay as they were in a given `out` [rows, N].  -> [rows, N]"""
    t = _lib.require_gpu(); L = _lib.lib()
    _check_matrix("x", x, 2)
    _check_matrix("w", w, 3, x.dtype, x.device)
    if transposed:
        w = w.transpose(1, 2)
    g, k, n = w.shape
    rows = x.shape[0]
    if x.shape[1] != k:
        raise ValueError(f"x has {x.shape[1]} columns, the weight blocks have {k} rows")
    if g < 1 or g > MAX_GROUPS or n < 1 or k < 1:
        raise ValueError(f"w: shape {tuple(w.shape)} is empty or has more than {MAX_GROUPS} groups")
    dtype = out.dtype if out is not None and out_dtype is None else out_dtype or x.dtype
    if dtype not in (x.dtype, t.float32):
        raise ValueError(f"out_dtype: {dtype} is neither {x.dtype} nor float32")
    flip, ldw, group_stride = _groups(w)
    off = offsets_device(offsets, g, rows, x.device)
    scale, shift = _affine("scale", scale, g, n, x.device), _affine("shift", shift, g, n, x.device)
    if scale is not None and shift is not None and scale.stride() != shift.stride():
        scale, shift = scale.contiguous(), shift.contiguous()
    some = scale if scale is not None else shift
    if some is not None and n > 1 and some.stride(1) != 1:
        scale, shift = (None if a is None else a.contiguous() for a in (scale, shift))
        some = scale if scale is not None else shift
    slope = float(slope)
    fill = out is None
    with t.cuda.device(x.device):
        if fill:
            out = _dev.empty((rows, n), dtype, x.device)
        else:
            _check_matrix("out", out, 2, dtype, x.device)
            if tuple(out.shape) != (rows, n):
                raise ValueError(f"out: shape {tuple(out.shape)}, expected {(rows, n)}")
            if any(_overlap(out, a) for a in (x, w)):
                raise ValueError("out: overlaps x or w")
        need = L.ct_grouped_product_workspace_bytes(_types()[x.dtype], rows, k, n, g)
        ws = _dev.workspace(need, x.device) if need else None
        _lib.check(L.ct_grouped_product(_types()[x.dtype], _types()[dtype], x.data_ptr(), _row_stride("x", x), rows, k, w.data_ptr(), group_stride, ldw,
                                        int(flip), n, off.data_ptr(), g, None if scale is None else scale.data_ptr(),
                                        None if shift is None else shift.data_ptr(), 0 if some is None or g == 1 else some.stride(0), slope, int(fill),
                                        out.data_ptr(), _row_stride("out", out), None if ws is None else ws.data_ptr(), need, _dev.stream(x.device)),
                   "ct_grouped_product")
    return out


def product_grad(dy, x, w, offsets, *, need_x: bool = True, need_w: bool = True, out_dtype=None):
    """The gradients of product(x, w, offsets) (no scale, shift or slope) for dy [rows, N] -> (dx [rows, K] of x's type, dw [G, K, N] of
    `out_dtype`: w's type, or float32); None in the place of one that is not needed.  Rows behind offsets[G] get a zero dx, a group without
    rows a zero dw[g].  Of a block that w.expand shares, each group's part comes separately: sum them."""
    t = _lib.require_gpu(); L = _lib.lib()
    _check_matrix("x", x, 2)
    _check_matrix("w", w, 3, x.dtype, x.device)
    _check_matrix("dy", dy, 2, x.dtype, x.device)
    g, k, n = w.shape
    rows = x.shape[0]
    if tuple(dy.shape) != (rows, n) or x.shape[1] != k:
        raise ValueError(f"dy {tuple(dy.shape)}, x {tuple(x.shape)} and w {tuple(w.shape)} do not fit each other")
    if g < 1 or g > MAX_GROUPS or n < 1 or k < 1:
        raise ValueError(f"w: shape {tuple(w.shape)} is empty or has more than {MAX_GROUPS} groups")
    dtype = out_dtype or w.dtype
    if dtype not in (w.dtype, t.float32):
        raise ValueError(f"out_dtype: {dtype} is neither {w.dtype} nor float32")
    off = offsets_device(offsets, g, rows, x.device)
    dx = product(dy, w, off, transposed=True) if need_x else None
    if not need_w:
        return dx, None
    with t.cuda.device(x.device):
        dw = _dev.empty((g, k, n), dtype, x.device)
        need = L.ct_grouped_product_dw_workspace_bytes(_types()[x.dtype], rows, k, n, g)
        ws = _dev.workspace(need, x.device) if need else None
        _lib.check(L.ct_grouped_product_dw(_types()[x.dtype], _types()[dtype], x.data_ptr(), _row_stride("x", x), rows, k, dy.data_ptr(),
                                           _row_stride("dy", dy), n, off.data_ptr(), g, dw.data_ptr(), k * n, n,
                                           None if ws is None else ws.data_ptr(), need, _dev.stream(x.device)), "ct_grouped_product_dw")
    return dx, dw
