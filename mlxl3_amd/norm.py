"""Root-mean-square norm of rows, with the residual's addition (``exl3_rms_norm`` of
``include/exl3_hip.h``): what stands in front of an attention block and of a feed-forward."""

from __future__ import annotations

from . import Exl3Error, _torch, load_library
from . import kv as _kv


def _laid(t):
    """(heads, token stride) of rows [..., width] that the kernel reads as they lie, or None:
    contiguous (heads 0: as others have them), or 2- and 3-dimensional with contiguous heads,
    tokens any distance apart."""
    if t.is_contiguous():
        return 0, t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return 1, t.stride(0)
    if t.dim() == 3 and _kv._rows_ok(t):
        return t.shape[1], t.stride(0)
    return None


def _floating(t, name: str):
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise Exl3Error(-1, f"{name} must be a device tensor")
    if t.dtype not in _kv._floats():
        raise Exl3Error(-1, f"{name} has dtype {t.dtype}, expected one of {tuple(_kv._FLOATS)}")
    return t


def _written(t, name: str, like, dtype):
    """A tensor that the kernel writes: like's shape and device, rows that it can write in place."""
    _floating(t, name)
    if t.shape != like.shape or (dtype is not None and t.dtype != dtype):
        raise Exl3Error(-1, f"{name} must have shape {tuple(like.shape)}" + (f" and dtype {dtype}" if dtype else ""))
    _kv._same(like.device, t, name)
    if _laid(t) is None:
        raise Exl3Error(-1, f"{name} must have contiguous rows")
    return t


def rms_norm(x, weight=None, eps: float = 1e-6, residual=None, total=None, out=None, dtype=None):
    """s / sqrt(mean(s^2) + eps) * weight over the last dimension of x [..., width] (f16, bf16 or
    f32), s = x, or x + residual.  weight [width] may be of another type, or None (ones).

    Without a residual the result, of x's type or `dtype`.  With one, of x's shape and of any of
    the types: (result, x + residual in the residual's type); `total` is where the sum goes -- the
    residual itself, or x: in place -- a new tensor by default.  The norm is taken of the sum before
    it is rounded.  `out`: where the result goes (may be x or the residual, where total is not).
    Tokens may lie any distance apart ([tokens, width], or [tokens, heads, width] with contiguous
    heads); x, residual and weight are copied where their strides are others.  Outputs and inputs
    that are not the same tensor do not overlap."""
    torch = _torch()
    x = _floating(x, "x")
    floats, device = _kv._FLOATS, x.device
    if x.dim() < 1 or x.shape[-1] < 1:
        raise Exl3Error(-1, f"norms take rows of at least one value, got shape {tuple(x.shape)}")
    if dtype is not None and dtype not in floats:
        raise Exl3Error(-1, f"unsupported norm output dtype {dtype}")
    try:
        eps = float(eps)
    except (TypeError, ValueError):
        raise Exl3Error(-1, f"norm eps must be a number, got {eps!r}") from None
    width = x.shape[-1]
    if weight is not None:
        _floating(weight, "weight")
        if tuple(weight.shape) != (width,):
            raise Exl3Error(-1, f"weight must have shape ({width},), got {tuple(weight.shape)}")
        _kv._same(device, weight, "weight")
        weight = weight.contiguous()
    if residual is None:
        if total is not None:
            raise Exl3Error(-1, "a sum needs a residual")
    else:
        _floating(residual, "residual")
        if residual.shape != x.shape:
            raise Exl3Error(-1, f"residual must have shape {tuple(x.shape)}, got {tuple(residual.shape)}")
        _kv._same(device, residual, "residual")
    if out is not None:
        _written(out, "out", x, dtype)
    if total is not None:
        _written(total, "total", x, residual.dtype)
        if total is out:
            raise Exl3Error(-1, "the sum and the norm are two outputs")
    if _laid(x) is None:
        x = x.contiguous()
    if residual is not None and _laid(residual) is None:
        residual = residual.contiguous()
    if out is None:
        out = torch.empty(x.shape, dtype=dtype or x.dtype, device=device)
    if residual is not None and total is None:
        total = torch.empty(x.shape, dtype=residual.dtype, device=device)
    if x.numel() == 0:
        return out if residual is None else (out, total)
    laid = [(0, 0) if t is None else _laid(t) for t in (x, residual, total, out)]
    heads = max(1, *(h for h, _ in laid))  # those that have gaps have x's
    xs, rs, ts, ys = (stride * heads if h == 0 else stride for h, stride in laid)
    _kv._launch(
        device, load_library().exl3_rms_norm, x.data_ptr(), floats[x.dtype], x.numel() // (width * heads), heads, width, xs,
        None if weight is None else weight.data_ptr(), 0 if weight is None else floats[weight.dtype], eps,
        None if residual is None else residual.data_ptr(), 0 if residual is None else floats[residual.dtype], rs,
        None if total is None else total.data_ptr(), ts, out.data_ptr(), floats[out.dtype], ys)
    return out if residual is None else (out, total)
