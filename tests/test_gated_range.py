"""The gated recurrence at the ends of its arguments' ranges. Oracle and counted bounds are those of ``test_gated.py``."""

import numpy as np
import pytest
import torch

import kla_b200
from test_gated import check, held, inputs, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("given,same", [([0, 40, 2 ** 32 + 40], [0, 40, 100]), ([0, 2 ** 31, 2 ** 31], [0, 100, 100]), ([0, 40, 2 ** 62], [0, 40, 100]),
                                        ([-2 ** 40, -2 ** 33 + 70, 100], [0, 0, 100]), ([2 ** 32, 2 ** 33], [100, 100])])
def test_bounds_past_32_bits_are_clamped(given, same):
    x, g = torch.randn(1, 100, 128, generator=torch.Generator("cuda").manual_seed(0), device="cuda").chunk(2, -1)
    got, want = (kla_b200.gated_scan_b200(x, g, cu_seqlens=torch.tensor(b, device="cuda")) for b in (given, same))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_state_written_in_place_is_known_to_autograd():
    x, g, state = torch.randn(3, 4, 64, device="cuda")
    weight = torch.randn(4, 64, device="cuda").requires_grad_()
    for written in (state, torch.empty_like(state)):
        before = written._version
        loss = (weight * written).sum()  # keeps `written` for weight's gradient
        with torch.no_grad():
            h, new = kla_b200.gated_step_b200(x, g, state, state_out=written)
        assert new.data_ptr() == written.data_ptr() and written._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    before = state._version
    kla_b200.gated_step_b200(x, g, state)
    assert state._version == before


def test_a_state_written_in_inference_mode():
    x, g, want = torch.randn(3, 4, 64, device="cuda")
    with torch.inference_mode():
        state = want.clone()
        _, new = kla_b200.gated_step_b200(x, g, want)
        for _ in range(2):
            state.copy_(want)
            kla_b200.gated_step_b200(x, g, state, state_out=state)
            assert torch.equal(state, new)
    with torch.no_grad():  # a tensor made there, written outside
        kla_b200.gated_step_b200(x, g, want, state_out=state)
    assert torch.equal(state, new)


def test_a_state_that_requires_a_gradient_is_not_written():
    x, g, state = torch.randn(3, 4, 64, device="cuda")
    leaf = torch.zeros(4, 64, device="cuda").requires_grad_()
    with pytest.raises(NotImplementedError):
        kla_b200.gated_step_b200(x, g, state, state_out=leaf)
    assert not leaf.any()
    with torch.no_grad():
        kla_b200.gated_step_b200(x, g, state, state_out=leaf)
    assert leaf.any()
