"""The gated feed-forward block under autocast with a residual stream of its own type. Oracle and bounds of ``test_mlp.py``."""

import pytest
import torch

import kla_b200
from test_mlp import HALF, NAMES, held, inputs, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [(130,), (2, 65), (10,), ()])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_a_residual_stream(dtype, lead):
    rows = max(1, int(torch.Size(lead).numel()))
    t, dy = inputs(rows, 64, 72, 64, bias=True)
    res = torch.randn(*lead, 64, generator=torch.Generator().manual_seed(3)).to(dtype).cuda().requires_grad_()
    leaves = {n: v.detach().float().requires_grad_() for n, v in t.items() if v is not None}
    given = {**leaves, "x": leaves["x"].view(*lead, 64), "residual": res}
    with torch.autocast("cuda", torch.bfloat16):
        y = kla_b200.gated_mlp_b200(**given)
        alone = kla_b200.gated_mlp_b200(**{**given, "residual": None})
    assert y.shape == (*lead, 64)
    if dtype == torch.bfloat16:
        assert y.dtype == torch.bfloat16
        want = oracle(*(t[n] for n in NAMES[:5]), res.detach().view(rows, 64), "silu", dy)
        held(y.view(rows, 64), want["y"], "y")
    else:
        assert y.dtype == torch.float32 and torch.equal(y, res.float() + alone.float())
        want = oracle(*(t[n] for n in NAMES), "silu", dy)
        # the block's result as it stands alone, and a rounding of the sum in float32
        off = (y.double() - res.double()).view(rows, 64) - want["y"].x
        assert (off.abs() <= want["y"].e + 2.0 ** -24 * y.double().abs().view(rows, 64)).all()
    grads = torch.autograd.grad(y, [*leaves.values(), res], dy.view(y.shape).to(y.dtype))
    for n, g in zip(leaves, grads):
        held(g.bfloat16(), want["d" + n], "d" + n)
    assert grads[-1].dtype == dtype
    assert ((grads[-1].double() - dy.double().view(grads[-1].shape)).abs() <= HALF * dy.double().abs().view(grads[-1].shape)).all()


@pytest.mark.parametrize("autocast", [True, False])
def test_residuals_that_do_not_fit_are_refused(autocast):
    t, _ = inputs(4, 16, 24, 16)
    with torch.autocast("cuda", torch.bfloat16, enabled=autocast):
        for res in (torch.zeros(3, 16), torch.zeros(4, 8), torch.zeros(16), torch.zeros(1, 4, 16)):
            with pytest.raises(ValueError):
                kla_b200.gated_mlp_b200(**{**t, "residual": res.cuda()})
        with pytest.raises(ValueError):
            kla_b200.gated_mlp_b200(**{**t, "residual": torch.zeros(4, 16)})
        with pytest.raises(NotImplementedError):
            kla_b200.gated_mlp_b200(**{**t, "residual": torch.zeros(4, 16, dtype=torch.float64, device="cuda")})
        if not autocast:
            with pytest.raises(NotImplementedError):
                kla_b200.gated_mlp_b200(**{**t, "residual": torch.zeros(4, 16, device="cuda")})
