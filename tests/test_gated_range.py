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
