"""A whole mixture-of-experts layer for a few tokens: router, SwiGLU experts in 4 or 8 bits, weighted sum.

The grouped dots (``ragged_dot_int4``) serve many rows sorted by expert; at decoding, with a handful of tokens, the
layer's time is the time to read the weights of the experts in use.  ``moe_swiglu`` takes the same weights and scales
as they are stored for the grouped dots and does everything from the tokens to their outputs on the device, with no
sorting, no padding to tiles and no host synchronisation.
"""
from __future__ import annotations

from typing import Any

from .metadata import GemmLayout, OperandDType, ScaleMode, ScaleSpec
from .native import DTYPE_CODES, LAYOUT_CODES, OUT_BF16, OUT_F32, moe_swiglu_on_device

MOE_MAX_TOKENS = 64
MOE_MAX_TOP_K = 16
MOE_MAX_EXPERTS = 1024
MOE_SIZE_MULTIPLE = 32  # the K of one int8 tensor-core instruction


def _torch() -> Any:
    try:
        import torch
    except ImportError as exc:  # pragma: no cover
        raise RuntimeError("torch is required for moe_swiglu") from exc
    return torch


def _check(torch: Any, name: str, tensor: Any, dtypes: tuple[Any, ...], shape: tuple[int, ...] | None, device: Any) -> None:
    if not isinstance(tensor, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not tensor.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and tensor.device != device:
        raise ValueError(f"{name} must be on {device}, the device of x; got {tensor.device}")
    if tensor.dtype not in dtypes:
        raise ValueError(f"{name} must have dtype {' or '.join(str(item) for item in dtypes)}; got {tensor.dtype}")
    if shape is not None and tensor.shape != shape:
        raise ValueError(f"{name} must have shape {shape}; got {tuple(tensor.shape)}")
    if not tensor.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if tensor.data_ptr() % 16 and name in _WIDE:
        raise ValueError(f"{name} must start on a multiple of 16 bytes")


_WIDE = frozenset(("x", "router_weight", "w_up_gate", "w_down", "up_gate_scale", "down_scale"))  # read 16 bytes at a time


def moe_swiglu(
    x: Any,
    w_up_gate: Any,
    w_down: Any,
    *,
    up_gate_scale: Any,
    down_scale: Any,
    router_weight: Any | None = None,
    top_k: int | None = None,
    topk_ids: Any | None = None,
    topk_weights: Any | None = None,
    renormalize: bool = True,
    dtype: OperandDType = OperandDType.INT4,
    layout: GemmLayout = GemmLayout.NN,
    scale: ScaleSpec = ScaleSpec(ScaleMode.PER_CHANNEL),
    return_routing: bool = False,
) -> Any:
    """``out[t] = sum_j p[t, j] * down_e(up_e(x[t]) * silu(gate_e(x[t])))`` over the ``top_k`` experts ``e`` of a token.

    ``x``: CUDA bfloat16 ``[T, H]``, up to 64 tokens.  ``w_up_gate``: ``[E, H/2, 2I]`` packed along K (INT4, NN), the up
    columns first, as ``fused_swiglu_up_gate`` and the grouped dots have them; ``[E, 2I, H/2]`` (NT); INT8 without the
    halving.  ``w_down``: ``[E, I/2, H]`` or ``[E, H, I/2]``.  Scales (bfloat16): per-channel ``up_gate_scale [E, 2I]``,
    ``down_scale [E, H]``; subchannel ``S``: ``[E, ceil(H/S), 2I]`` and ``[E, ceil(I/S), H]``.  ``H`` and ``I`` are
    multiples of 32.

    Routing: ``router_weight [E, H]`` (bfloat16 or float32) and ``top_k``: the largest logits, ties to the lowest expert and
    NaN below all others, weighted with their softmax (``renormalize=False``: the softmax over all experts).  Or
    ``topk_ids [T, k]`` (int32 or int64) and ``topk_weights [T, k]`` (float32) from elsewhere; they are not read on the host,
    and an id outside ``[0, E)``, as -1, stands for no expert.  ``return_routing=True`` returns
    ``(out, topk_ids, topk_weights)``.

    The tokens, and the activations between the two products, are quantised as ``quantize_tokens`` does (the
    activations without being rounded before).  Integer sums are exact, the choice of experts and the border cases of
    the quantiser are decided in float64, an expert's result is rounded to float32, weighted and added up in the order of
    the choices, and the sum is rounded to bfloat16: the same bits on every run.  With one scale a column also whatever
    other tokens are in the call; with K-group scales the float64 sums of the second product are divided by the number of
    experts in use, and a last bit may hang on that.  No autograd.
    """
    torch = _torch()
    if type(dtype) is not OperandDType:
        raise TypeError(f"dtype must be an OperandDType, got {type(dtype).__name__}")
    if type(layout) is not GemmLayout:
        raise TypeError(f"layout must be a GemmLayout, got {type(layout).__name__}")
    if layout not in (GemmLayout.NN, GemmLayout.NT):
        raise ValueError(f"moe_swiglu supports layouts nn and nt; got {layout.value}")
    _check(torch, "x", x, (torch.bfloat16,), None, None)
    if x.ndim != 2:
        raise ValueError(f"x must have shape (T, H); got {tuple(x.shape)}")
    tokens, hidden = int(x.shape[0]), int(x.shape[1])
    if tokens > MOE_MAX_TOKENS:
        raise ValueError(f"x must have at most {MOE_MAX_TOKENS} tokens; got {tokens} (use ragged_dot_int4 for more rows)")
    code_type = (torch.uint8,) if dtype is OperandDType.INT4 else (torch.int8,)
    device = x.device
    _check(torch, "w_up_gate", w_up_gate, code_type, None, device)
    if w_up_gate.ndim != 3:
        raise ValueError(f"w_up_gate must be a grouped tensor; got shape {tuple(w_up_gate.shape)}")
    nn = layout is GemmLayout.NN
    experts, columns = int(w_up_gate.shape[0]), int(w_up_gate.shape[2 if nn else 1])
    inner = columns // 2
    if columns % 2 or hidden % MOE_SIZE_MULTIPLE or inner % MOE_SIZE_MULTIPLE or not hidden or not inner:
        raise ValueError(f"H and I must be multiples of {MOE_SIZE_MULTIPLE}; got H={hidden} and {columns} up/gate columns")
    if not 0 < experts <= MOE_MAX_EXPERTS:
        raise ValueError(f"there must be 1 to {MOE_MAX_EXPERTS} experts; got {experts}")
    per_byte = 2 if dtype is OperandDType.INT4 else 1
    kb, ib = hidden // per_byte, inner // per_byte
    if tuple(w_up_gate.shape) != ((experts, kb, columns) if nn else (experts, columns, kb)):
        raise ValueError(f"w_up_gate does not match H={hidden} for layout={layout.value}; got shape {tuple(w_up_gate.shape)}")
    _check(torch, "w_down", w_down, code_type, (experts, ib, hidden) if nn else (experts, hidden, ib), device)
    sub = scale.subchannel_size or 0
    bf16 = (torch.bfloat16,)
    _check(torch, "up_gate_scale", up_gate_scale, bf16, (experts, -(-hidden // sub), columns) if sub else (experts, columns), device)
    _check(torch, "down_scale", down_scale, bf16, (experts, -(-inner // sub), hidden) if sub else (experts, hidden), device)

    if router_weight is not None:
        if topk_ids is not None or topk_weights is not None:
            raise ValueError("give either router_weight and top_k or topk_ids and topk_weights, not both")
        if isinstance(top_k, bool) or not isinstance(top_k, int):
            raise TypeError("top_k must be a Python int")
        _check(torch, "router_weight", router_weight, (torch.bfloat16, torch.float32), (experts, hidden), device)
        if return_routing:
            topk_ids = torch.empty((tokens, max(top_k, 0)), device=device, dtype=torch.int32)
            topk_weights = torch.empty((tokens, max(top_k, 0)), device=device, dtype=torch.float32)
    else:
        if topk_ids is None or topk_weights is None:
            raise ValueError("give either router_weight and top_k or topk_ids and topk_weights")
        _check(torch, "topk_ids", topk_ids, (torch.int32, torch.int64), None, device)
        if topk_ids.ndim != 2 or int(topk_ids.shape[0]) != tokens:
            raise ValueError(f"topk_ids must have shape ({tokens}, k); got {tuple(topk_ids.shape)}")
        _check(torch, "topk_weights", topk_weights, (torch.float32,), tuple(topk_ids.shape), device)
        if top_k is not None and top_k != int(topk_ids.shape[1]):
            raise ValueError(f"top_k is {top_k} but topk_ids has {int(topk_ids.shape[1])} columns")
        top_k = int(topk_ids.shape[1])
    if not 0 < top_k <= min(MOE_MAX_TOP_K, experts):
        raise ValueError(f"top_k must be in [1, {min(MOE_MAX_TOP_K, experts)}]; got {top_k}")
    if tokens == 0:
        out = torch.empty_like(x)
    else:
        fields = (
            DTYPE_CODES[dtype], LAYOUT_CODES[layout], sub, tokens, hidden, inner, experts, top_k,
            OUT_F32 if router_weight is not None and router_weight.dtype is torch.float32 else OUT_BF16, int(bool(renormalize)),
            64 if topk_ids is not None and topk_ids.dtype is torch.int64 else 32)
        out = moe_swiglu_on_device(
            fields, x, router_weight=router_weight, topk_ids=topk_ids, topk_weights=topk_weights, w_up_gate=w_up_gate,
            up_gate_scale=up_gate_scale, w_down=w_down, down_scale=down_scale)
    return (out, topk_ids, topk_weights) if return_routing else out
