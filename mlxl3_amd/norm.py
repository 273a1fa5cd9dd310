"""Root-mean-square norm of rows, with the residual's addition (``exl3_rms_norm`` of
``include/exl3_hip.h``): what stands in front of an attention block and of a feed-forward."""

from __future__ import annotations

from . import Exl3Error, _torch, load_library
from .kv import _floats, _launch, _rows_ok, _same


def _laid(t):
    """(heads, token stride) of rows [..., width] that the kernel reads as they lie, or None:
    contiguous (heads 0: as others have them), or 2- and 3-dimensional with contiguous heads,
    tokens any distance apart."""
    if t.is_contiguous():
        return 0, t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return 1, t.stride(0)
    if t.dim() == 3 and _rows_ok(t):
        return t.shape[1], t.stride(0)
    return None


def _code(t, name: str) -> int:
    """The type's code of a floating device tensor."""
    torch, floats = _torch(), _floats()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise Exl3Error(-1, f"{name} must be a device tensor")
    code = floats.get(t.dtype)
    if code is None:
        raise Exl3Error(-1, f"{name} has dtype {t.dtype}, expected one of {tuple(floats)}")
    return code


def _written(t, name: str, shape, device, dtype) -> int:
    """The type's code of a tensor that the kernel writes: rows that it can write in place."""
    code = _code(t, name)
    if t.shape != shape or (dtype is not None and t.dtype != dtype):
        raise Exl3Error(-1, f"{name} must have shape {tuple(shape)}" + (f" and dtype {dtype}" if dtype else ""))
    _same(device, t, name)
    if _laid(t) is None:
        raise Exl3Error(-1, f"{name} must have contiguous rows")
    return code


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
    x_code = _code(x, "x")
    shape, device = x.shape, x.device
    width = shape[-1] if shape else 0
    if not 0 < width < 2**31:
        raise Exl3Error(-1, f"norms take rows of at least one value and fewer than 2^31, got shape {tuple(shape)}")
    if type(eps) is not float:
        try:
            eps = float(eps)
        except (TypeError, ValueError):
            raise Exl3Error(-1, f"norm eps must be a number, got {eps!r}") from None
    w_code = r_code = 0
    if weight is not None:
        w_code = _code(weight, "weight")
        if weight.dim() != 1 or weight.numel() != width:
            raise Exl3Error(-1, f"weight must have shape ({width},), got {tuple(weight.shape)}")
        _same(device, weight, "weight")
        weight = weight.contiguous()
    if residual is not None:
        r_code = _code(residual, "residual")
        if residual.shape != shape:
            raise Exl3Error(-1, f"residual must have shape {tuple(shape)}, got {tuple(residual.shape)}")
        _same(device, residual, "residual")
    elif total is not None:
        raise Exl3Error(-1, "a sum needs a residual")
    if out is not None:
        y_code = _written(out, "out", shape, device, dtype)
    elif dtype is None or dtype == x.dtype:
        y_code = x_code
    else:
        y_code = _floats().get(dtype)
        if y_code is None:
            raise Exl3Error(-1, f"unsupported norm output dtype {dtype}")
    if total is not None:
        _written(total, "total", shape, device, residual.dtype)
        if total is out:
            raise Exl3Error(-1, "the sum and the norm are two outputs")
    # (heads, token stride) of x, residual, total and out where one of them has gaps
    laid = None
    if not (x.is_contiguous() and (residual is None or residual.is_contiguous())
            and (total is None or total.is_contiguous()) and (out is None or out.is_contiguous())):
        laid = [(0, width) if t is None else _laid(t) for t in (x, residual, total, out)]
        if laid[0] is None:
            x, laid[0] = x.contiguous(), (0, width)
        if laid[1] is None:
            residual, laid[1] = residual.contiguous(), (0, width)
    if out is None:
        out = torch.empty_like(x, dtype=dtype, memory_format=torch.contiguous_format)
    if residual is not None and total is None:
        total = torch.empty_like(residual, memory_format=torch.contiguous_format)
    count = x.numel()
    if count == 0:
        return out if residual is None else (out, total)
    heads, xs, rs, ts, ys = 1, width, width, width, width
    if laid is not None:
        heads = max(1, max(laid)[0])  # those that have gaps have x's
        if heads >= 2**31:
            raise Exl3Error(-1, f"norms take fewer than 2^31 heads, got {heads}")
        xs, rs, ts, ys = (stride if h else stride * heads for h, stride in laid)
    _launch(
        device, load_library().exl3_rms_norm, x.data_ptr(), x_code, count // (width * heads), heads, width, xs,
        None if weight is None else weight.data_ptr(), w_code, eps,
        None if residual is None else residual.data_ptr(), r_code, rs,
        None if total is None else total.data_ptr(), ts, out.data_ptr(), y_code, ys)
    return out if residual is None else (out, total)
