"""The gated recurrence on the B200 kernels, beside the raw affine scan (``affine_scan_b200``):

    h_t = a_t h_{t-1} + (1 - a_t) x_t,   a_t = sigmoid(gate_t),   h_{-1} = initial_state (zeros when None)

channel by channel. Where ``affine_scan_b200`` takes materialised float32 coefficients and starts from zero, this forms them
from gates on the way, in float32 whatever the activations' type, takes a batch of sequences or packed sequences of different
lengths, starts from states and returns the states it ends in, and spreads few or long sequences over the GPU. Differentiable
with respect to ``x``, ``gate`` and ``initial_state``. ``gated_step_b200`` is one token of it. There is no CPU or eager path:
what the kernels do not take raises ``NotImplementedError``.
"""

from __future__ import annotations

import torch

from . import _lib


def gated_scan_b200(x: torch.Tensor, gate: torch.Tensor, initial_state: torch.Tensor | None = None,
                    cu_seqlens: torch.Tensor | None = None):
    """``(h, state)``: ``h`` like ``x``, ``state`` float32 ``[sequences, D]``, the value behind every sequence's last step.

    ``x``, ``gate``: ``[B, L, D]`` float32 or bfloat16, any strides with adjacent channels (others are copied), such as the
    halves of one projection. ``initial_state``: float32 ``[sequences, D]``. ``cu_seqlens``: bounds of packed sequences,
    ``[sequences + 1]`` int32 (int64 is converted) on the device, ``x`` being ``[1, L, D]``: sequence ``n`` is the rows
    ``cu_seqlens[n]`` to ``cu_seqlens[n + 1]``; the bounds must not decrease, which is not checked (values outside ``[0, L]``
    are clamped). A sequence without rows leaves the state it started from; rows that belong to no sequence get zeros, in
    ``h`` and in the gradients. Where gates forget, what they leave of a state (and of its gradient) has the relative accuracy of
    ``sigmoid(gate)``: 2^-14 in float32 and 2^-11 in bfloat16 at least. An infinite state stays infinite, unless an infinity of
    the other sign or a gate whose ``sigmoid`` is 0 in float32 (below -87) makes it NaN; so does an infinite gradient of it."""
    return _lib.host().gated_scan(x, gate, initial_state, cu_seqlens)


def gated_step_b200(x: torch.Tensor, gate: torch.Tensor, state: torch.Tensor, state_out: torch.Tensor | None = None):
    """One token: ``(h, new_state)`` for ``x``, ``gate`` ``[B, D]`` and ``state`` float32 ``[B, D]``. ``state_out`` receives the
    new state where it is given, and may be ``state`` itself (a captured token then advances it with every replay): an
    in-place operation like torch's own. No backward."""
    return _lib.host().gated_step(x, gate, state, state_out)
