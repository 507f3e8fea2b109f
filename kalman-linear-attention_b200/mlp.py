"""The gated feed-forward block on the B200 kernels:

    y = (act(x Wg^T + bg) * (x Wu^T + bu)) W3^T + b3 (+ residual),    w12 = [Wg; Wu]

which is the swiglu MLP of a block of the reference's ``SequenceModel`` (src/kla/layers/common.py:99-122) for ``act = silu``,
differentiable with respect to everything it is given. Both first projections, their biases, the activation and the product are
one kernel on the tensor cores; so are the second projection, its bias and the residual sum. The backward has no elementwise pass of
its own either: the gradients of gate and up are formed where the gradient of their product is. bfloat16, accumulated in float32.
For the few rows of decoded tokens in inference the projections are the decode kernels (``kla_b200_linear``). There is no CPU or
eager path: what the kernels do not take raises ``NotImplementedError``.
"""

from __future__ import annotations

import torch

from . import _lib


def gated_mlp_b200(x: torch.Tensor, w12: torch.Tensor, w3: torch.Tensor, b12: torch.Tensor | None = None, b3: torch.Tensor | None = None,
                   residual: torch.Tensor | None = None, activation: str | None = "silu") -> torch.Tensor:
    """``x`` ``[..., d]``, ``w12`` ``[2 H, d]`` (gate's rows, then up's), ``w3`` ``[out, H]``, ``b12`` ``[2 H]``, ``b3`` ``[out]``,
    ``residual`` ``[..., out]`` added to the result in float32 before it is rounded. ``activation``: ``"silu"``, ``"gelu"`` (the exact
    one), ``"relu"`` or None. Any sizes and strides: rows that are not 16-byte aligned (a width that is no multiple of 8) are copied
    first. Under a bfloat16 autocast float32 and float16 ``x``, weights and biases are converted as ``F.linear`` does; a ``residual`` of
    those types is not, but added to the rounded bfloat16 result as ``residual + F.linear(...)`` would be, and the sum is float32.

    A call that is to be differentiated keeps ``x``, the weights and three ``[rows, H]`` tensors of 16 bits for the backward: the
    product, and gate and up with nine bits of mantissa over 2^-31 to 2^32 (beyond, their gradients are NaN; but a gate that large
    and negative under silu, gelu or relu takes no part, whatever its size: a hidden unit may be masked by its bias)."""
    wide = None  # a residual the sum with which is float32
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
        if residual is not None and residual.dtype in (torch.float32, torch.float16) and residual.device == x.device and x.dim() > 0:
            if residual.shape != (*x.shape[:-1], w3.shape[0] if w3.dim() == 2 else -1):
                raise ValueError("kla_b200: residual has the output's shape")
            wide, residual = residual, None
        x, w12, w3, b12, b3 = (t.to(torch.bfloat16) if t is not None and t.is_cuda and t.dtype in (torch.float32, torch.float16) else t
                               for t in (x, w12, w3, b12, b3))
    lead = None
    if x.dim() != 2:
        if x.dim() == 0:
            raise ValueError("kla_b200: x is [..., d]")
        lead = x.shape[:-1]
        if residual is not None:
            if residual.dim() == 0 or residual.shape[:-1] != lead:
                raise ValueError("kla_b200: residual has the output's shape")
            residual = residual.reshape(lead.numel(), residual.shape[-1])
        x = x.reshape(lead.numel(), x.shape[-1])
    y = _lib.host().gated_mlp(x, w12, w3, b12, b3, residual, activation)
    if lead is not None:
        y = y.view(*lead, y.shape[-1])
    return y if wide is None else wide.float() + y
