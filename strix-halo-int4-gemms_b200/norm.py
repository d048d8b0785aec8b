"""Layer norm around the quantised products: forward, backward, and fused with the quantiser.

The reference has no norms; a model built on its products takes them from elsewhere and quantises the result with
a constant scale (``quant.py:14-29``).  Here the norm can hand its rows to the products directly
(:func:`layer_norm_quantize`), and a training step has both directions as explicit functions, in the manner of
``ragged_dot_int4`` and ``ragged_dot_int4_bwd``: no autograd.
"""
from __future__ import annotations

import math
from typing import Any

from .metadata import OperandDType, ScaleMode, ScaleSpec
from .native import layer_norm_bwd_on_device, layer_norm_on_device, layer_norm_quantize_on_device
from .quant import _code_bits

DEFAULT_EPS = 1e-5
FLOAT32_NONE, FLOAT32_MOST = 2.0 ** -150, (2.0 - 2.0 ** -23) * 2.0 ** 127  # what rounds to zero, and the largest


def _torch() -> Any:
    try:
        import torch
    except ImportError as exc:  # pragma: no cover
        raise RuntimeError("torch is required for layer_norm") from exc
    return torch


def _check_values(torch: Any, name: str, tensor: Any, dtypes: tuple[Any, ...]) -> None:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if tensor.dtype not in dtypes:
        names = " or ".join(str(item) for item in dtypes)
        raise ValueError(f"{name} must have dtype {names}; got {tensor.dtype}")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_norm_operands(torch: Any, x: Any, weight: Any, bias: Any | None) -> None:
    types = (torch.bfloat16, torch.float32)
    _check_values(torch, "x", x, types)
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must have at least one value a row; got shape {tuple(x.shape)}")
    cols = int(x.shape[-1])
    for name, tensor in (("weight", weight), ("bias", bias)):
        if tensor is None and name == "bias":
            continue
        _check_values(torch, name, tensor, types)
        if tensor.shape != (cols,):
            raise ValueError(f"{name} must have shape ({cols},); got {tuple(tensor.shape)}")
        if tensor.device != x.device:
            raise ValueError(f"{name} must be on {x.device}, the device of x; got {tensor.device}")
    if bias is not None and bias.dtype != weight.dtype:
        raise ValueError(f"bias must have the dtype of weight, {weight.dtype}; got {bias.dtype}")


def _check_eps(eps: float) -> float:
    if isinstance(eps, bool) or not isinstance(eps, (int, float)):
        raise TypeError("eps must be a Python int or float scalar")
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError("eps must be finite and non-negative")
    return float(eps)


def layer_norm(x: Any, weight: Any, bias: Any | None = None, *, eps: float = DEFAULT_EPS) -> tuple[Any, Any, Any]:
    """``(y, mean, rstd)``: ``y = (x - mean) * rstd * weight + bias`` over the last axis.

    ``x``: CUDA bfloat16 or float32 ``[..., N]``, contiguous; ``y`` has its dtype.  ``weight`` and ``bias`` (or
    None) ``[N]``, bfloat16 or float32, whatever ``x`` is.  ``mean`` and ``rstd = 1 / sqrt(var + eps)`` are float32
    ``[...]``, what :func:`layer_norm_bwd` needs.  Statistics in float32, the mean in two parts, so that its rounding shifts no
    row (equal values give the bias); one rounding of ``y`` at the end.  ``eps`` is zero or a number that float32 has room for.
    """
    torch = _torch()
    _check_norm_operands(torch, x, weight, bias)
    eps = _check_eps(eps)
    if eps != 0.0 and not FLOAT32_NONE < eps <= FLOAT32_MOST:  # it is added to a float32 variance
        raise ValueError("eps must be zero or within the range of float32")
    return layer_norm_on_device(x, weight, bias, eps=eps)


def layer_norm_quantize(
    x: Any,
    weight: Any,
    bias: Any | None = None,
    *,
    eps: float = DEFAULT_EPS,
    dtype: OperandDType = OperandDType.INT4,
    scale: ScaleSpec = ScaleSpec(ScaleMode.PER_CHANNEL),
) -> tuple[Any, Any]:
    """``(codes, scales)``: :func:`layer_norm` and ``quantize_tokens`` in one pass, the A operand of the products.

    Operands as :func:`layer_norm`, results as ``quantize_tokens``.  The norm is not rounded before it is quantised
    (the two calls one after the other round it to ``x.dtype`` in between), and each code and scale is that of the
    exactly computed norm: a value next to the border of two codes is settled in float64.
    """
    torch = _torch()
    bits = _code_bits(dtype)
    _check_norm_operands(torch, x, weight, bias)
    return layer_norm_quantize_on_device(x, weight, bias, eps=_check_eps(eps), bits=bits, subchannel=scale.subchannel_size or 0)


def layer_norm_bwd(dy: Any, x: Any, weight: Any, mean: Any, rstd: Any) -> tuple[Any, Any, Any]:
    """``(dx, dweight, dbias)`` of :func:`layer_norm`.

    ``dy`` has the shape and dtype of ``x``; ``mean`` and ``rstd`` are the forward pass's.  ``dx`` has the dtype of
    ``x``; ``dweight`` and ``dbias`` are float32 ``[N]``, as the products' weight gradients are, summed over all rows
    in a fixed order (the same bits on every run; zeros where there are no rows).
    """
    torch = _torch()
    _check_norm_operands(torch, x, weight, None)
    _check_values(torch, "dy", dy, (x.dtype,))
    if dy.shape != x.shape or dy.device != x.device:
        raise ValueError(f"dy must have the shape and device of x, {tuple(x.shape)} on {x.device}; got {tuple(dy.shape)} on {dy.device}")
    for name, tensor in (("mean", mean), ("rstd", rstd)):
        _check_values(torch, name, tensor, (torch.float32,))
        if tensor.shape != x.shape[:-1] or tensor.device != x.device:
            raise ValueError(f"{name} must have shape {tuple(x.shape[:-1])} on {x.device}; got {tuple(tensor.shape)} on {tensor.device}")
    return layer_norm_bwd_on_device(dy, x, weight, mean, rstd)
