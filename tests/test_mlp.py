"""The gated feed-forward block against float64: forward, backward, sizes that divide into nothing, a token's few rows.

Tolerances are counted, not chosen: ``oracle`` carries a bound beside every value. A product of n terms accumulated in float32
is off by at most (n + 2) 2^-23 of the sum of its terms' absolute values (an addition of the tensor core may truncate: a whole
step of 2^-23); what is rounded to bfloat16 on the way (h, and in the backward dg, du) by 2^-8 of itself; g and u, kept for the
backward with nine bits of mantissa, by 2^-10 of themselves and 2^-41; the activation's
exponential and reciprocal by 2^-20. Errors go through products by their absolute values. Slopes: |silu'| and |gelu'| are below
1.13, |silu''| and |gelu''| below 0.8; relu's slope is undetermined where g is within its own error of zero.
"""

import ctypes
import importlib
import threading

import pytest
import torch
import torch.nn.functional as F

import kla_b200

lib = importlib.import_module("kalman-linear-attention_b200._lib")
ACTS = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu, None: lambda t: t}
HALF, STEP = 2.0 ** -8, 2.0 ** -23


class V:
    """A value with a bound of its error."""

    def __init__(self, x, e=None):
        self.x, self.e = x, torch.zeros_like(x) if e is None else e

    def t(self):
        return V(self.x.t(), self.e.t())

    def __add__(self, o):
        return V(self.x + o.x, self.e + o.e)

    def __mul__(self, o):
        return V(self.x * o.x, self.x.abs() * o.e + self.e * o.x.abs() + self.e * o.e)

    def __matmul__(self, o):
        a, b = self.x.abs() + self.e, o.x.abs() + o.e
        exact = a @ b - self.x.abs() @ o.x.abs()  # what the operands' errors make of the sum at most
        return V(self.x @ o.x, exact + (self.x.shape[1] + 2) * STEP * (a @ b))

    def rounded(self):
        return V(self.x, self.e + HALF * (self.x.abs() + self.e))

    def kept(self):
        return V(self.x, self.e + 2.0 ** -10 * (self.x.abs() + self.e) + 2.0 ** -41)


def oracle(x, w12, w3, b12, b3, residual, act, dy):
    d64 = lambda t: None if t is None else V(t.detach().double().cuda())  # noqa: E731
    x, w12, w3, b12, b3, residual, dy = map(d64, (x, w12, w3, b12, b3, residual, dy))
    H = w3.x.shape[1]
    gu = x @ w12.t()
    if b12 is not None:
        gu = gu + b12
    half = lambda v, i: V(v.x[:, i * H:(i + 1) * H], v.e[:, i * H:(i + 1) * H])  # noqa: E731
    g, u = half(gu, 0), half(gu, 1)

    def f(g, slope):
        with torch.enable_grad():
            leaf = g.x.clone().requires_grad_()
            val = ACTS[act](leaf)
            der, = torch.autograd.grad(val.sum(), leaf)
        if not slope:
            return V(val.detach(), 1.13 * g.e + 2.0 ** -20 * (val.detach().abs() + g.e))
        if act == "relu":
            return V(der, (g.x.abs() <= g.e).double())
        return V(der, torch.zeros_like(der) if act is None else 0.8 * g.e + 2.0 ** -20 * (1 + g.x.abs()))

    h = (f(g, False) * u).rounded()
    y = h @ w3.t()
    for more in (b3, residual):
        if more is not None:
            y = y + more
    out = {"y": y.rounded()}
    if dy is None:
        return out
    gs, us = g.kept(), u.kept()
    dh = dy @ w3
    dg, du = (dh * us * f(gs, True)).rounded(), (dh * f(gs, False)).rounded()
    dgu = V(torch.cat((dg.x, du.x), 1), torch.cat((dg.e, du.e), 1))
    ones = V(torch.ones(1, x.x.shape[0], dtype=torch.float64, device="cuda"))
    out.update(dx=(dgu @ w12).rounded(), dw12=(dgu.t() @ x).rounded(), dw3=(dy.t() @ h).rounded(), db12=(ones @ dgu).rounded(), db3=(ones @ dy).rounded(),
               dresidual=dy)
    return out


def held(got, want, what):
    assert got.dtype == torch.bfloat16 and got.shape == want.x.reshape(got.shape).shape
    ratio = (got.detach().double() - want.x.reshape(got.shape)).abs() / (want.e.reshape(got.shape) + 1e-37)
    assert torch.isfinite(got).all() and (got.numel() == 0 or ratio.max() <= 1.0), f"{what}: {ratio.max():.2f} of its tolerance"


def inputs(rows, d, H, out, bias=False, residual=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).bfloat16().cuda()  # noqa: E731
    return dict(x=rn(rows, d), w12=rn(2 * H, d, scale=d ** -0.5), w3=rn(out, H, scale=H ** -0.5), b12=rn(2 * H, scale=0.5) if bias else None,
                b3=rn(out) if bias else None, residual=rn(rows, out) if residual else None), rn(rows, out)


NAMES = ("x", "w12", "w3", "b12", "b3", "residual")


def check(t, dy, act="silu"):
    want = oracle(*(t[n] for n in NAMES), act, dy)
    with torch.no_grad():
        held(kla_b200.gated_mlp_b200(**t, activation=act), want["y"], "y in inference")
    names = [n for n in NAMES if t[n] is not None]
    leaves = [t[n].detach().requires_grad_() for n in names]
    y = kla_b200.gated_mlp_b200(**{**t, **dict(zip(names, leaves))}, activation=act)
    held(y, want["y"], "y")
    for n, got in zip(names, torch.autograd.grad(y, leaves, dy)):
        assert got.shape == t[n].shape
        held(got, want["d" + n], "d" + n)


def test_the_oracles_gradients_are_differences():
    torch.manual_seed(0)
    rows, d, H, out, step = 3, 4, 5, 2, 1e-5
    t = [torch.randn(*s, dtype=torch.float64) for s in ((rows, d), (2 * H, d), (out, H), (2 * H,), (out,))]
    dy = torch.randn(rows, out, dtype=torch.float64)

    def loss(x, w12, w3, b12, b3):
        g, u = F.linear(x, w12, b12).chunk(2, -1)
        return (F.linear(F.silu(g) * u, w3, b3) * dy).sum()

    g, u = F.linear(t[0], t[1], t[3]).chunk(2, -1)
    s = torch.sigmoid(g)
    dh, h = dy @ t[2], g * s * u
    dgu = torch.cat((dh * u * s * (1 + g * (1 - s)), dh * g * s), 1)
    for i, want in enumerate((dgu @ t[1], dgu.t() @ t[0], dy.t() @ h, dgu.sum(0), dy.sum(0))):
        for j in range(t[i].numel()):
            v = []
            for sign in (step, -step):
                args = [a.clone() for a in t]
                args[i].view(-1)[j] += sign
                v.append(loss(*args))
            # third derivatives of order 10 times step^2, and 2^-53 / step of sums of order 10
            assert abs((v[0] - v[1]) / (2 * step) - want.reshape(-1)[j]) < 1e-8


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d,H,out", [
    (128, 64, 64, 64), (1, 8, 8, 8), (2, 1, 1, 1), (5, 3, 7, 5), (129, 65, 130, 72), (300, 136, 200, 120), (64, 8, 1000, 264),
    (257, 768, 264, 768), (700, 512, 1365, 512), (4096, 192, 768, 192), (9000, 128, 72, 128)])
def test_forward_and_backward(rows, d, H, out):
    check(*inputs(rows, d, H, out))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
@pytest.mark.parametrize("rows,d,H,out", [(200, 96, 136, 96), (77, 33, 45, 31), (3, 64, 64, 64)])
def test_activations_biases_and_residual(act, rows, d, H, out):
    check(*inputs(rows, d, H, out, bias=True, residual=True), act=act)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 8, 16, 17, 32, 33])
@pytest.mark.parametrize("bias", [False, True])
def test_few_rows(rows, bias):
    check(*inputs(rows, 256, 688, 256, bias=bias, residual=True))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d,H,out", [(1000, 328, 2721, 72), (1000, 2400, 2721, 64)])
def test_tiles_of_96_columns_of_gate_and_up(rows, d, H, out):
    """Sizes that tiles of 128 columns would leave in a second round of CTAs."""
    check(*inputs(rows, d, H, out, bias=True))


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("rows,d,H,out", [(33, 64, 5456, 200), (64, 512, 2731, 511), (1, 100, 4000, 36), (257, 330, 6001, 67), (130, 1024, 5456, 1024)])
def test_few_rows_of_long_sums_are_split(rows, d, H, out, bias):
    assert lib.load().kla_b200_mlp_fwd_work_bytes(ctypes.byref(lib.MlpArgs(rows=rows, d=d, H=H, out=out))) >= 2 * 4 * rows * out
    check(*inputs(rows, d, H, out, bias=bias, residual=bias), act="gelu" if bias else "silu")


@pytest.mark.gpu
def test_leading_dimensions_strides_and_broadcast_gradients():
    t, _ = inputs(6 * 50, 64, 96, 40, residual=True)
    want = oracle(*(t[n] for n in NAMES), "silu", torch.ones(300, 40))
    x = torch.zeros(6, 50, 80, device="cuda", dtype=torch.bfloat16)[..., 8:72]  # rows 160 bytes apart, 16-byte aligned
    x.copy_(t["x"].view(6, 50, 64))
    w12 = t["w12"].t().contiguous().t()  # columns adjacent: copied
    res = t["residual"].view(6, 50, 40).transpose(0, 1).contiguous().transpose(0, 1)
    leaves = [v.detach().requires_grad_() for v in (x, w12, t["w3"], res)]
    y = kla_b200.gated_mlp_b200(leaves[0], leaves[1], leaves[2], residual=leaves[3])
    assert y.shape == (6, 50, 40)
    held(y, want["y"], "y")
    for n, got in zip(("dx", "dw12", "dw3", "dresidual"), torch.autograd.grad(y.sum(), leaves)):
        held(got, want[n], n)
    one = kla_b200.gated_mlp_b200(x[0, 0], t["w12"], t["w3"], residual=res[0, 0])
    assert one.shape == (40,)
    held(one, V(want["y"].x[0], want["y"].e[0]), "one row")


@pytest.mark.gpu
def test_only_the_gradients_that_are_wanted():
    t, dy = inputs(150, 64, 72, 64, bias=True)
    full = None
    for wanted in (NAMES[:5], *((n,) for n in NAMES[:5]), ("w12", "b3")):
        given = {n: (v.detach().requires_grad_() if n in wanted else v) for n, v in t.items()}
        y = kla_b200.gated_mlp_b200(**given)
        got = dict(zip(wanted, torch.autograd.grad(y, [given[n] for n in wanted], dy)))
        full = full or got
        assert all(torch.equal(got[n], full[n]) for n in wanted)


@pytest.mark.gpu
def test_a_second_derivative_raises():
    t, _ = inputs(20, 16, 24, 16, residual=True)
    x = t["x"].requires_grad_()
    y = kla_b200.gated_mlp_b200(**t)
    dx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.gpu
def test_a_broadcast_residual():
    t, dy = inputs(40, 64, 72, 64)
    row = torch.randn(64, device="cuda").bfloat16().requires_grad_()
    t["residual"] = row.expand(40, 64)
    want = oracle(*(t[n] for n in NAMES), "silu", dy)
    y = kla_b200.gated_mlp_b200(**t)
    held(y, want["y"], "y")
    got, = torch.autograd.grad(y, row, dy)
    assert torch.equal(got, torch.autograd.grad(row.expand(40, 64), row, dy)[0])


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused_not_dropped():
    from torch.autograd import forward_ad

    t, _ = inputs(8, 16, 24, 16)
    x = torch.randn(1, 8, 16, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t["w3"], torch.ones_like(t["w3"]))
        with pytest.raises(NotImplementedError):
            kla_b200.gated_mlp_b200(**{**t, "w3": dual})
        gate = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            kla_b200.gated_scan_b200(x, gate)
        with pytest.raises(NotImplementedError):
            kla_b200.gated_step_b200(x[0], gate[0], x[0].clone())


@pytest.mark.gpu
def test_no_rows():
    t, dy = inputs(0, 16, 24, 16, bias=True)
    leaves = {n: v.detach().requires_grad_() for n, v in t.items() if v is not None}
    y = kla_b200.gated_mlp_b200(**leaves)
    assert y.shape == (0, 16)
    for n, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
        assert g.shape == leaves[n].shape and not g.any()


@pytest.mark.gpu
def test_autocast_converts_as_linear_does():
    t, dy = inputs(130, 64, 72, 64, bias=True)
    leaves = {n: v.detach().float().requires_grad_() for n, v in t.items() if v is not None}
    with torch.autocast("cuda", torch.bfloat16):
        y = kla_b200.gated_mlp_b200(**leaves)
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    want = oracle(*(t[n] for n in NAMES), "silu", dy)
    held(y, want["y"], "y")
    for n, g in zip(leaves, grads):
        assert g.dtype == torch.float32
        held(g.bfloat16(), want["d" + n], "d" + n)


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_rows():
    t, _ = inputs(300, 64, 96, 64)
    y0 = kla_b200.gated_mlp_b200(**t)
    t["x"][7, 3] = float("nan")
    t["x"][200, 0] = float("inf")
    y = kla_b200.gated_mlp_b200(**t)
    bad = ~torch.isfinite(y).all(1)
    assert bad[[7, 200]].all() and bad.sum() == 2 and torch.equal(y[~bad], y0[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0 ** -30, 2.0 ** -12, 2.0 ** 12])
def test_scales_of_gate_and_up(scale):
    """The kept gate and up hold their accuracy over the range that is documented."""
    t, dy = inputs(140, 64, 72, 64)
    t["x"] *= scale
    check(t, dy, act=None)


@pytest.mark.gpu
def test_gate_and_up_beyond_the_kept_range_have_nan_gradients():
    t, dy = inputs(140, 64, 72, 64)
    t["x"][3] *= 2.0 ** 40
    given = {**t, "x": t["x"].detach().requires_grad_()}
    y = kla_b200.gated_mlp_b200(**given, activation=None)
    dx, = torch.autograd.grad(y, given["x"], dy)
    assert torch.isfinite(y).all() and torch.isnan(dx[3]).any()
    keep = torch.arange(140) != 3
    assert torch.isfinite(dx[keep]).all()


@pytest.mark.gpu
def test_captured_on_another_stream_and_the_same_every_time():
    t, dy = inputs(1500, 128, 344, 128, bias=True)
    leaves = {n: v.detach().requires_grad_() for n, v in t.items() if v is not None}

    def step():
        y = kla_b200.gated_mlp_b200(**leaves)
        return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), dy))

    want = [v.clone() for v in step()]
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(on_side, want))
    for _ in range(2):
        for v in got:
            v.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_a_new_threads_first_call():
    """Its memory comes from the allocator's cache, so nothing before the call has bound the device's context to the thread."""
    t, _ = inputs(300, 64, 96, 64)
    y0 = kla_b200.gated_mlp_b200(**t)
    del_me = kla_b200.gated_mlp_b200(**t)
    torch.cuda.synchronize()
    del del_me  # what the thread's call takes
    got = []
    thread = threading.Thread(target=lambda: got.append(kla_b200.gated_mlp_b200(**t)))
    thread.start()
    thread.join()
    assert len(got) == 1 and torch.equal(got[0], y0)


@pytest.mark.gpu
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right():
    L = lib.load()
    t, _ = inputs(300, 512, 96, 64)
    y0 = kla_b200.gated_mlp_b200(**t)
    assert lib.device_status() == 0
    try:
        assert L.kla_b200_test_hooks(3_000_000, 2) == 0  # 3 ms; the loader stops in front of its third block
        kla_b200.gated_mlp_b200(**t)
        st = lib.device_status()
    finally:
        assert L.kla_b200_test_hooks(0, -1) == 0
    # the products wait for the block (0x41), the epilogue for them (0x43)
    assert st & 0x100 and (st & 0xFF) in (0x41, 0x43), hex(st)
    assert torch.equal(kla_b200.gated_mlp_b200(**t), y0) and lib.device_status() == 0


def mlp_refusals():
    t, _ = inputs(4, 16, 24, 16, bias=True, residual=True)
    call = lambda **kw: lambda: kla_b200.gated_mlp_b200(**{**t, **kw})  # noqa: E731
    return [
        (NotImplementedError, call(x=t["x"].float())),
        (NotImplementedError, call(x=t["x"].half(), w12=t["w12"].half(), w3=t["w3"].half())),
        (NotImplementedError, call(b12=t["b12"].float())),
        (ValueError, call(x=t["x"][:, :8])),
        (ValueError, call(x=t["x"][0, 0])),
        (ValueError, call(w12=t["w12"][:46])),
        (ValueError, call(w12=t["w12"][0])),
        (ValueError, call(w3=t["w3"][:, :23])),
        (ValueError, call(b12=t["b12"][:24])),
        (ValueError, call(b3=t["b3"][:8])),
        (ValueError, call(residual=t["residual"][:3])),
        (ValueError, call(residual=t["residual"][:, :8])),
        (ValueError, call(activation="tanh")),
        (ValueError, call(w3=t["w3"].cpu())),
    ]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(14))
def test_refusals(i):
    error, call = mlp_refusals()[i]
    with pytest.raises(error):
        call()


def test_cpu_tensors_are_refused():
    x, w12, w3 = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((4, 16), (48, 16), (16, 24)))
    for given in ((x, w12, w3), (x.requires_grad_(), w12, w3)):
        with pytest.raises(NotImplementedError):
            kla_b200.gated_mlp_b200(*given)


def test_entry_points_reject_bad_arguments_without_cuda():
    L = lib.load()
    full = dict(rows=4, d=16, H=24, out=16, x=64, w12=64, w3=64, h=64, y=64, x_stride=16, w12_stride=16, w3_stride=24, h_stride=24, y_stride=16,
                gu=64, gu_stride=48, dgu=64, dy=64, dy_stride=16, dx=64, dx_stride=16, dw12=64, dw3=64, work=64)
    A = lambda **kw: ctypes.byref(lib.MlpArgs(**{**full, **kw}))  # noqa: E731
    for fn in (L.kla_b200_mlp_fwd, L.kla_b200_mlp_bwd):
        assert fn(None, None) == 1
        assert fn(A(rows=-1), None) == 1 and fn(A(d=0), None) == 1
        assert fn(A(activation=4), None) == 1
        assert fn(A(rows=1 << 31), None) == 2
        assert fn(A(w3=None), None) == 1 and fn(A(w3=72), None) == 4
        assert fn(A(w3_stride=16), None) == 1 and fn(A(w3_stride=28), None) == 4
        assert fn(A(x_stride=20), None) == 4 and fn(A(h=None), None) == 1
        assert fn(A(gu_stride=56), None) == 4
    assert L.kla_b200_mlp_fwd(A(rows=0), None) == 0
    assert L.kla_b200_mlp_fwd(A(y_stride=8), None) == 1 and L.kla_b200_mlp_fwd(A(residual=65, residual_stride=16), None) == 4
    assert L.kla_b200_mlp_bwd(A(work=None), None) == 1 and L.kla_b200_mlp_bwd(A(dw3=72), None) == 4 and L.kla_b200_mlp_bwd(A(dx_stride=8), None) == 1
    assert L.kla_b200_mlp_work_bytes(A(rows=0)) == 0 and L.kla_b200_mlp_work_bytes(None) == 0
    assert L.kla_b200_mlp_work_bytes(A()) >= 4 * 2 * 24  # the row sums of gate's and up's gradients
