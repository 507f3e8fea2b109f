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


U = 2.0 ** -24
FORGET = {torch.float32: -6.0, torch.bfloat16: -8.0}  # below, a step is taken by a itself


def relative_oracle(x, g, h0, dh, dend, forget):
    """As ``test_gated.oracle`` for a batch, with bounds relative to what a step leaves: where a gate forgets, a is off by 2^-21 + 2^-24 |g| of
    itself (its exponential, a reciprocal, the argument's rounding), z by that share of a, and up to eight roundings are of
    a |h| and |x|; where it holds they are of |h| and |x|, and z's error is z's share of either. hm, um: the recurrences of absolute
    values, which no composed map exceeds."""
    B, L, D = x.shape
    z, a = 1 / (1 + np.exp(g)), 1 / (1 + np.exp(-g))
    dz = 2.0 ** -21 + U * np.minimum(np.abs(g), 104.0)
    f = g < forget

    def step(t, e, hm, xa):
        return a[:, t] * e + np.where(f[:, t], a[:, t] * (dz[:, t] + 8 * U) * hm + (a[:, t] * dz[:, t] + 8 * U) * xa,
                                      z[:, t] * dz[:, t] * (hm + xa) + 8 * U * (hm + xa))

    h, hm, e = h0.copy(), np.abs(h0), np.zeros_like(h0)
    hs, es = [], []
    for t in range(L):
        e = step(t, e, hm, np.abs(x[:, t]))
        h, hm = a[:, t] * h + z[:, t] * x[:, t], a[:, t] * hm + z[:, t] * np.abs(x[:, t])
        hs.append(h), es.append(e)
    u, um, ue = dend.copy(), np.abs(dend), np.zeros_like(dend)
    for t in reversed(range(L)):
        c, cm = dh[:, t] + u, np.abs(dh[:, t]) + um
        ue = step(t, ue + U * cm, cm, 0.0)
        u, um = a[:, t] * c, a[:, t] * cm
    return (np.stack(hs, 1), np.stack(es, 1)), (hs[-1], es[-1]), (u, ue)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread,keep", [(0.5, -16.0), (3.0, -6.0), (0.5, -30.0), (20.0, -20.0), (2.0, 2.0)])
@pytest.mark.parametrize("B,L,D", [(2, 1, 64), (1, 2, 5), (3, 3, 66), (2, 70, 8), (1, 700, 64)])
def test_what_gates_leave_when_they_forget(B, L, D, spread, keep, dtype):
    """Without input a state, and without gradients of h the gradient of the state a sequence starts from, is a product of a's."""
    both, h0, dh, dend = inputs(B, L, D, B, dtype, spread=spread, keep=keep)
    gen = torch.Generator().manual_seed(1)
    silent = torch.rand(B, L, D, generator=gen) < 0.9
    silent[:, :, ::2] = True
    x = both[..., :D].clone()
    x[silent], dh[silent.flip(1)] = 0.0, 0.0
    g = both[..., D:]
    leaves = [t.cuda().requires_grad_() for t in (x, g, h0)]
    h, end = kla_b200.gated_scan_b200(*leaves)
    _, _, dstate = torch.autograd.grad((h, end), leaves, (dh.cuda(), dend.cuda()))
    want = relative_oracle(*(t.double().numpy() for t in (x, g, h0, dh, dend)), FORGET[dtype])
    for got, (value, bound), what in zip((h, end, dstate), want, ("h", "end", "dstate")):
        held(got, value, bound, what)
    one, state = kla_b200.gated_step_b200(x[:, 0].cuda(), g[:, 0].cuda(), h0.cuda())
    held(one, want[0][0][:, 0], want[0][1][:, 0], "token")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread,keep", [(0.5, 9.0), (0.5, -9.0), (4.0, -4.0), (30.0, 0.0)])
@pytest.mark.parametrize("layout", ["halves", "dense"])
def test_gates_that_hold_and_forget_of_either_type(spread, keep, dtype, layout):
    check(2, 700, 48, dtype, spread=spread, keep=keep, layout=layout)
    check(1, 900, 67, dtype, spread=spread, keep=keep, layout=layout, bounds=[0, 3, 3, 400, 401, 890])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_neighbours_do_not_change_a_channels_bits(dtype):
    """The choice between the two ways of taking a tile is a warp's; a channel whose gates hold gets the same either way."""
    both, h0, dh, dend = (t.cuda() for t in inputs(2, 200, 64, 2, dtype))
    got = []
    for shut in (False, True):
        g = both[..., 64:].clone()
        g[..., :64] = g[..., :64].clamp_min(-2.5)
        if shut:
            g[:, ::7, 5] = -12.0
        leaves = [t.detach().requires_grad_() for t in (both[..., :64], g, h0)]
        h, end = kla_b200.gated_scan_b200(*leaves)
        got.append((h, end, *torch.autograd.grad((h, end), leaves, (dh, dend))))
    others = torch.arange(64, device="cuda") != 5
    for name, a, b in zip(("h", "end", "dx", "dgate", "dstate"), *got):
        assert torch.equal(a[..., others], b[..., others]), name


def same_kinds(got, want, what):
    got = got.detach().double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN"
    assert np.array_equal(np.where(np.isinf(got), got, 0.0), np.where(np.isinf(want), want, 0.0)), f"{what}: infinities"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread,keep", [(1.0, 2.0), (1.5, -1.0), (1.0, -6.0)])
@pytest.mark.parametrize("B,L,D,bounds", [(2, 300, 24, None), (1, 2500, 24, None), (3, 70, 65, None), (1, 900, 24, [0, 40, 41, 41, 700, 880]), (2, 1, 24, None)])
def test_infinite_values_are_taken_as_the_formula_takes_them(B, L, D, bounds, spread, keep, dtype):
    """a inf is inf while a is not 0: inputs, states and gradients that are infinite leave infinite values behind, of their sign; NaN
    comes of infinities that meet with opposite signs and of a gate that leaves nothing. Other channels keep their bits."""
    n = B if bounds is None else len(bounds) - 1
    both, h0, dh, dend = inputs(B, L, D, n, dtype, spread=spread, keep=keep)
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    inf, i, j = float("inf"), L // 3, 2 * L // 3
    runs = []
    for broken in (False, True):
        x, g, s, d, e = both[..., :D].clone(), both[..., D:].clone(), h0.clone(), dh.clone(), dend.clone()
        if broken:
            x[:, i, 0] = inf
            x[:, L - 1, 1] = -inf
            s[:, 2] = inf
            x[:, i, 3], x[:, j, 3] = inf, -inf
            d[:, j, 4] = inf
            e[:, 5] = -inf
            x[:, i, 6], g[:, j, 6] = inf, -inf
            x[:, i, 7], g[:, i, 7] = -inf, -inf
            d[:, j, 8], d[:, i, 8] = inf, -inf
            s[:, 9], d[:, j, 9] = -inf, inf
            x[:, i, 10], g[:, j, 10] = inf, inf
        leaves = [t.cuda().requires_grad_() for t in (x, g, s)]
        h, end = kla_b200.gated_scan_b200(*leaves, cu_seqlens=cu)
        runs.append((h, end, *torch.autograd.grad((h, end), leaves, (d.cuda(), e.cuda()))))
    with np.errstate(all="ignore"):
        want, _ = oracle(*(t.double().numpy() for t in (x, g, s)), bounds, d.double().numpy(), e.double().numpy())
    for name, clean, got in zip(("h", "end", "dx", "dgate", "dstate"), *runs):
        same_kinds(got, want[name], name)
        assert torch.equal(got[..., 11:], clean[..., 11:]), name
    with np.errstate(all="ignore"):
        first, _ = oracle(*(t.double().numpy() for t in (x[:, :1], g[:, :1], s[:B])))
    token, state = kla_b200.gated_step_b200(leaves[0].detach()[:, 0], leaves[1].detach()[:, 0], leaves[2].detach()[:B].contiguous())
    same_kinds(token, first["h"][:, 0], "token")
    same_kinds(state, first["end"], "state")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L,D", [(300, 64), (400, 1024), (700, 256), (1000, 1536), (2000, 64), (2500, 2048)])
def test_a_lone_packed_sequence_is_taken_as_a_batch_of_one(L, D, dtype):
    """The same CTAs share it: the same bits."""
    both, h0, dh, dend = (t.cuda() for t in inputs(1, L, D, 1, dtype))
    got = []
    for cu in (None, torch.tensor([0, L], dtype=torch.int32, device="cuda")):
        leaves = [t.detach().requires_grad_() for t in (both[..., :D], both[..., D:], h0)]
        h, end = kla_b200.gated_scan_b200(*leaves, cu_seqlens=cu)
        got.append((h, end, *torch.autograd.grad((h, end), leaves, (dh, dend))))
    for name, a, b in zip(("h", "end", "dx", "dgate", "dstate"), *got):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L,bounds", [(300, None), (2500, None), (900, [0, 40, 41, 41, 700, 880]), (1, None)])
def test_nan_reaches_what_the_formula_takes_it_to(L, bounds, dtype):
    D, i = 24, L // 3
    n = 1 if bounds is None else len(bounds) - 1
    both, h0, dh, dend = inputs(1, L, D, n, dtype)
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    runs, nan = [], float("nan")
    for broken in (False, True):
        x, g, s, d, e = both[..., :D].clone(), both[..., D:].clone(), h0.clone(), dh.clone(), dend.clone()
        if broken:
            x[:, i, 0] = nan
            g[:, i, 1] = nan
            s[:, 2] = nan
            d[:, i, 3] = nan
            e[:, 4] = nan
        leaves = [t.cuda().requires_grad_() for t in (x, g, s)]
        h, end = kla_b200.gated_scan_b200(*leaves, cu_seqlens=cu)
        runs.append((h, end, *torch.autograd.grad((h, end), leaves, (d.cuda(), e.cuda()))))
    with np.errstate(all="ignore"):
        want, _ = oracle(*(t.double().numpy() for t in (x, g, s)), bounds, d.double().numpy(), e.double().numpy())
    for name, clean, got in zip(("h", "end", "dx", "dgate", "dstate"), *runs):
        same_kinds(got, want[name], name)
        assert torch.equal(got[..., 5:], clean[..., 5:]), name
