"""What the gated feed-forward block's gradients are where gate and up leave the range they are kept in, and beside NaN and
infinity. The oracle and its counted bounds are those of ``test_mlp.py``."""

import pytest
import torch

import kla_b200
from test_mlp import NAMES, held, inputs, oracle

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(torch.bfloat16).min


def gradients(t, dy, act):
    names = [n for n in NAMES if t[n] is not None]
    leaves = [t[n].detach().requires_grad_() for n in names]
    y = kla_b200.gated_mlp_b200(**{**t, **dict(zip(names, leaves))}, activation=act)
    return y, dict(zip(names, torch.autograd.grad(y, leaves, dy)))


@pytest.mark.parametrize("act,mask", [("silu", LOWEST), ("gelu", LOWEST), ("relu", LOWEST), ("relu", -float("inf")), ("silu", -2.0 ** 34)])
@pytest.mark.parametrize("rows,d,H,out", [(140, 64, 72, 64), (300, 33, 333, 48)])
def test_a_masked_hidden_unit(act, mask, rows, d, H, out):
    """A unit whose gate a bias closes takes no part: the others' results are those of the block without it, its own gradients 0."""
    t, dy = inputs(rows, d, H, out, bias=True)
    masked = torch.arange(0, H, 5)
    t["b12"][masked] = mask
    units = torch.ones(H, dtype=torch.bool)
    units[masked] = False
    both = units.repeat(2)
    want = oracle(t["x"], t["w12"][both.cuda()], t["w3"][:, units.cuda()], t["b12"][both.cuda()], t["b3"], None, act, dy)
    y, grads = gradients(t, dy, act)
    held(y, want["y"], "y")
    for n, axis, some in (("x", None, None), ("w12", 0, both), ("w3", 1, units), ("b12", 0, both), ("b3", None, None)):
        got = grads[n]
        if some is None:
            held(got, want["d" + n], "d" + n)
        else:
            held(got.index_select(axis, some.nonzero().squeeze(1).cuda()), want["d" + n], "d" + n)
            assert not got.index_select(axis, (~some).nonzero().squeeze(1).cuda()).any(), n


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
def test_nan_and_infinity_stay_in_their_rows_of_dx(act):
    """The rows' sums are sums over all rows: NaN there."""
    t, dy = inputs(300, 64, 96, 64, bias=True)
    _, clean = gradients(t, dy, act)
    t["x"][7, 3] = float("nan")
    t["x"][200, 0] = float("inf")
    _, grads = gradients(t, dy, act)
    bad = ~torch.isfinite(grads["x"]).all(1)
    assert bad[[7, 200]].all() and bad.sum() == 2 and torch.equal(grads["x"][~bad], clean["x"][~bad])
    assert torch.isnan(grads["w12"]).any() and torch.isnan(grads["b12"]).any() and torch.equal(grads["b3"], clean["b3"])
    dy = dy.clone()
    t, _ = inputs(300, 64, 96, 64, bias=True)
    dy[5, 5] = float("nan")
    _, grads = gradients(t, dy, act)
    assert torch.isnan(grads["x"][5]).all() and torch.isnan(grads["b3"][5]) and torch.isfinite(grads["b3"][6:]).all()
    keep = torch.arange(300) != 5
    assert torch.equal(grads["x"][keep], clean["x"][keep])


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_a_gate_of_minus_infinity_is_nan_as_torchs_is(act):
    t, dy = inputs(140, 64, 72, 64, bias=True)
    t["b12"][3] = -float("inf")
    y, grads = gradients(t, dy, act)
    assert torch.isnan(y).all() and torch.isnan(grads["x"]).all() and torch.isnan(grads["w12"][3]).all()


@pytest.mark.parametrize("scale", [2.0 ** -40, 2.0 ** -33, 2.0 ** -32, 2.0 ** -31, 2.0 ** -30, 1.0, 2.0 ** 31])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_the_kept_range_and_its_steps(scale, sign):
    """One row whose gates lie just short of half a step, from where du's rounding goes the same way: nine bits of mantissa down to
    2^-31, steps of 2^-40 below. Gates are a weight and a bias, which adds bits that bfloat16 does not have."""
    H = 8
    fine = sign * scale * torch.tensor([2.0 ** -8 - 2.0 ** -11, 2.0 ** -9 - 2.0 ** -12, 2.0 ** -10 - 2.0 ** -13, 2.0 ** -10, 0.0, 2.0 ** -12, 2.0 ** -7, 2.0 ** -8])
    t = dict(x=torch.eye(1, 8), w12=torch.zeros(2 * H, 8), w3=torch.full((1, H), 1 - 2.0 ** -8), b12=torch.cat((fine, torch.zeros(H))), b3=None, residual=None)
    t["w12"][:H, 0], t["w12"][H:, 0] = sign * scale, 1.0
    t = {n: None if v is None else v.bfloat16().cuda() for n, v in t.items()}
    dy = torch.full((1, 1), 1 + 2.0 ** -7).bfloat16().cuda()  # dh = 1 + 2^-8 - 2^-15
    want = oracle(*(t[n] for n in NAMES), None, dy)
    _, grads = gradients(t, dy, None)
    held(grads["w12"], want["dw12"], "dw12")
    held(grads["b12"], want["db12"], "db12")


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
def test_the_oracle_itself_is_differences(act):
    """``test_mlp.oracle``'s own values, for every activation, with biases and residual."""
    gen = torch.Generator().manual_seed(2)
    rows, d, H, out, step = 3, 4, 5, 2, 1e-5
    sizes = dict(x=(rows, d), w12=(2 * H, d), w3=(out, H), b12=(2 * H,), b3=(out,), residual=(rows, out))
    t = {n: torch.randn(*sizes[n], generator=gen, dtype=torch.float64) for n in NAMES}
    dy = torch.randn(rows, out, generator=gen, dtype=torch.float64)
    want = oracle(*t.values(), act, dy)
    gu = t["x"] @ t["w12"].T + t["b12"]
    assert act != "relu" or gu[:, :H].abs().min() > 100 * step  # no difference crosses the kink
    loss = lambda given: (oracle(*given.values(), act, None)["y"].x.cpu() * dy).sum().item()  # noqa: E731
    for n in NAMES:
        for i in range(t[n].numel()):
            v = []
            for sign in (step, -step):
                moved = {k: a.clone() for k, a in t.items()}
                moved[n].view(-1)[i] += sign
                v.append(loss(moved))
            # third derivatives of order 10 times step^2, and 2^-53 / step of sums of order 10
            assert abs((v[0] - v[1]) / (2 * step) - want["d" + n].x.reshape(-1)[i].item()) < 1e-8, (n, i)
