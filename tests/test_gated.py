"""The gated recurrence against a sequential restatement in float64: forward, backward, packed sequences, one token.

Tolerances are counted along the recurrence, not chosen: ``oracle`` carries, beside every value, a bound of how far a float32
evaluation may be off. A gate's z = sigmoid(-g) comes from an exponential and a reciprocal of the hardware (2 ulp = 2^-22 each)
of an argument g log2(e) that is rounded (2^-24 |g| in the exponential), so z is off by DZ(g) = 2^-21 + 2^-24 |g| of itself.
A step adds z DZ (|x| + |h|) for that and roundings of 2^-24 of its terms: two of its own, and up to six where stretches are
composed as maps (the products A and their application lose 2^-24 a step each, of at most the values' size).
"""

import ctypes
import importlib

import numpy as np
import pytest
import torch

import kla_b200

lib = importlib.import_module("kalman-linear-attention_b200._lib")
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # a rounding's largest relative error


def spans(B, L, bounds):
    return [(b, 0, L) for b in range(B)] if bounds is None else [(0, lo, hi) for lo, hi in zip(bounds[:-1], bounds[1:])]


def oracle(x, g, h0, bounds=None, dh=None, dend=None):
    """Values and bounds by name, from float64 arrays [B, L, D] (h0, dend [sequences, D])."""
    B, L, D = x.shape
    seqs = spans(B, L, bounds)
    z, a = 1 / (1 + np.exp(g)), 1 / (1 + np.exp(-g))
    dz = 2.0 ** -21 + U * np.minimum(np.abs(g), 104.0)  # beyond, the exponential is 0 or inf in float32 and z exact
    out = {k: np.zeros_like(x) for k in ("h", "dx", "dgate")}
    err = {k: np.zeros_like(x) for k in out}
    for k in ("end", "dstate"):
        out[k], err[k] = np.zeros((len(seqs), D)), np.zeros((len(seqs), D))
    for n, (b, lo, hi) in enumerate(seqs):
        h, e = h0[n].copy(), np.zeros(D)
        big = np.abs(h) + (np.abs(x[b, lo:hi]).max(0) if hi > lo else 0.0)  # no value is larger
        before, before_e = [], []
        for t in range(lo, hi):
            before.append(h), before_e.append(e)
            e = a[b, t] * e + z[b, t] * dz[b, t] * (np.abs(x[b, t]) + np.abs(h)) + 8 * U * big
            h = a[b, t] * h + z[b, t] * x[b, t]
            out["h"][b, t], err["h"][b, t] = h, e
        out["end"][n], err["end"][n] = h, e
        if dh is None:
            continue
        u, ue = dend[n].copy(), np.zeros(D)
        um = np.abs(u)  # the recurrence of the absolute values: no sum or composed map of it is larger
        for t in range(hi - 1, lo - 1, -1):
            c, cm = dh[b, t] + u, np.abs(dh[b, t]) + um
            ce = ue + U * cm
            at, zt = a[b, t], z[b, t]
            hb, hbe = before[t - lo], before_e[t - lo]
            d, s = hb - x[b, t], np.abs(hb) + np.abs(x[b, t])
            out["dx"][b, t], err["dx"][b, t] = zt * c, zt * (ce + np.abs(c) * (dz[b, t] + 2 * U))
            out["dgate"][b, t] = c * d * zt * at
            err["dgate"][b, t] = zt * at * (ce * s + np.abs(c) * hbe + np.abs(c) * s * (2 * dz[b, t] + 6 * U))
            ue = at * ce + zt * dz[b, t] * np.abs(c) + 8 * U * cm
            u, um = at * c, at * cm
        out["dstate"][n], err["dstate"][n] = u, ue
    return out, err


def held(got, want, bound, what):
    """got within the bound and, for its type, one rounding of want."""
    g = got.detach().double().cpu().numpy()
    tol = bound + HALF[got.dtype] * (np.abs(want) + bound) + 1e-37
    worst = np.max(np.abs(g - want) / tol) if g.size else 0.0
    assert np.isfinite(g).all() and worst <= 1.0, f"{what}: {worst:.2f} of its tolerance"


def inputs(B, L, D, n, dtype, seed=0, spread=1.5, keep=2.0):
    """Input and gate as halves of one projection, state, and the gradients that come in."""
    gen = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    both = torch.cat((rn(B, L, D), spread * rn(B, L, D) + keep), dim=-1).to(dtype)
    return both, rn(n, D), rn(B, L, D).to(dtype), rn(n, D)


def check(B, L, D, dtype, carry=True, bounds=None, seed=0, layout="halves", **kw):
    n = B if bounds is None else len(bounds) - 1
    both, h0, dh, dend = inputs(B, L, D, n, dtype, seed, **kw)
    cu = None if bounds is None else torch.tensor(bounds, dtype=torch.int32, device="cuda")
    both = both.cuda()
    x, g = both[..., :D], both[..., D:]
    if layout == "dense":
        x, g = x.contiguous(), g.contiguous()
    elif layout == "time first":
        x, g = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (x, g))
    elif layout == "channels apart":
        x, g = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (x, g))
    state = h0.cuda() if carry else None
    leaves = [t.detach().requires_grad_() for t in (x, g, *((state,) if carry else ()))]
    h, end = kla_b200.gated_scan_b200(*leaves, cu_seqlens=cu)
    grads = torch.autograd.grad((h, end), leaves, (dh.cuda(), dend.cuda()))
    with torch.no_grad():
        h_inf, end_inf = kla_b200.gated_scan_b200(x, g, state, cu_seqlens=cu)
    assert torch.equal(h, h_inf) and torch.equal(end, end_inf)
    f64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    want, err = oracle(f64(x), f64(g), f64(h0) if carry else np.zeros((n, D)), bounds, f64(dh), f64(dend))
    assert h.dtype == dtype and end.dtype == torch.float32 and grads[0].dtype == dtype
    held(h, want["h"], err["h"], "h")
    held(end, want["end"], err["end"], "end")
    for name, got in zip(("dx", "dgate", "dstate"), grads):
        held(got, want[name], err[name], name)


def test_the_oracles_gradients_are_differences():
    rng = np.random.default_rng(0)
    bounds, L, D = [0, 3, 3, 9], 9, 2
    x, g, h0 = rng.standard_normal((1, L, D)), rng.standard_normal((1, L, D)), rng.standard_normal((3, D))
    dh, dend = rng.standard_normal((1, L, D)), rng.standard_normal((3, D))

    def loss(x, g, h0):
        o, _ = oracle(x, g, h0, bounds)
        return (o["h"] * dh).sum() + (o["end"] * dend).sum()

    want, _ = oracle(x, g, h0, bounds, dh, dend)
    step = 1e-5
    for i, name in enumerate(("dx", "dgate", "dstate")):
        args = [x, g, h0]
        for at in np.ndindex(args[i].shape):
            up, down = args[i].copy(), args[i].copy()
            up[at] += step
            down[at] -= step
            d = (loss(*args[:i], up, *args[i + 1:]) - loss(*args[:i], down, *args[i + 1:])) / (2 * step)
            # third derivatives of order 1 times step^2, and 2^-53 / step of sums of order 10
            assert abs(d - want[name][at]) < 1e-9, (name, at)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (2, 1, 64), (3, 7, 5), (2, 63, 64), (1, 64, 66), (2, 65, 63), (1, 129, 130), (2, 700, 33),
                                   (1, 2500, 8), (40, 70, 384)])
def test_forward_and_backward(B, L, D, dtype):
    check(B, L, D, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["dense", "time first", "channels apart"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(layout, dtype):
    check(3, 130, 70, dtype, layout=layout, carry=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bounds", [[0, 200], [0, 0, 1, 1, 64, 129, 193, 200], [0, 130, 130], [5, 70, 180], [0, 0, 0], [0]])
def test_packed_sequences(bounds, dtype):
    check(1, 200, 67, dtype, bounds=bounds)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_packed_sequences_share_clusters(dtype):
    """Few sequences, one of them most of the rows, others of one row and none; thousands of rows that belong to no sequence."""
    check(1, 18000, 40, dtype, bounds=[300, 11001, 11002, 11002, 13500])


@pytest.mark.gpu
def test_bounds_outside_the_rows_are_clamped():
    check_against = lambda b: kla_b200.gated_scan_b200(  # noqa: E731
        *torch.randn(1, 100, 128, generator=torch.Generator("cuda").manual_seed(0), device="cuda").chunk(2, -1),
        cu_seqlens=torch.tensor(b, device="cuda"))
    for got, want in ((check_against([-7, 40, 1000]), check_against([0, 40, 100])), (check_against([200, 300]), check_against([100, 100]))):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("spread,keep", [(0.5, 9.0), (0.5, -9.0), (30.0, 0.0)])
def test_gates_that_hold_and_gates_that_forget(spread, keep):
    check(2, 1500, 16, torch.float32, spread=spread, keep=keep)


@pytest.mark.gpu
def test_infinite_gates_and_nan():
    x, g, s = torch.randn(1, 300, 64).cuda(), torch.zeros(1, 300, 64).cuda(), torch.randn(1, 64).cuda()
    g[:, 100:] = float("inf")  # hold
    g[:, 200] = -float("inf")  # take the input as it is
    h, end = kla_b200.gated_scan_b200(x, g, s)
    with np.errstate(over="ignore"):
        want, err = oracle(*(t.double().cpu().numpy() for t in (x, g, s)))
    held(h, want["h"], err["h"], "h")  # a held value changes by the roundings of the maps in front of a warp's steps only
    assert np.array_equal(want["h"][:, 100:200], want["h"][:, 99:100].repeat(100, 1))
    assert torch.equal(h[:, 200:], x[:, 200:201].expand(-1, 100, -1)) and torch.equal(end, x[:, 200])
    g[:, 150, 3] = float("nan")
    x[:, 20, 5] = float("nan")
    h2, _ = kla_b200.gated_scan_b200(x, g, s)
    bad = torch.isnan(h2)
    assert bad[:, 150:, 3].all() and bad[:, 20:200, 5].all() and bad.sum() == 150 + 280
    keep = torch.ones(64, dtype=torch.bool)
    keep[[3, 5]] = False
    assert torch.equal(h2[..., keep.cuda()], h[..., keep.cuda()])


@pytest.mark.gpu
def test_empty_sizes():
    for shape in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        x = torch.randn(shape, device="cuda").requires_grad_()
        s = torch.randn(shape[0], shape[2], device="cuda").requires_grad_()
        h, end = kla_b200.gated_scan_b200(x, x.detach() * 0, s)
        assert h.shape == shape and (shape[1] or torch.equal(end, s))
        dx, ds = torch.autograd.grad((h.sum() + 2 * end.sum()), (x, s))
        assert dx.shape == shape and (shape[1] or torch.equal(ds, torch.full_like(s, 2.0)))
    h, s = kla_b200.gated_step_b200(*torch.randn(2, 0, 8, device="cuda"), torch.zeros(0, 8, device="cuda"))
    assert h.shape == s.shape == (0, 8)


@pytest.mark.gpu
def test_gradients_of_one_output_alone_and_of_broadcast_gradients():
    both, h0, _, dend = (t.cuda() for t in inputs(2, 150, 64, 2, torch.float32))
    x, g, s = (t.detach().requires_grad_() for t in (both[..., :64], both[..., 64:], h0))
    h, end = kla_b200.gated_scan_b200(x, g, s)
    zero, one = torch.zeros_like(h), torch.ones_like(h)
    for outs, full in (((end,), (zero, dend)), ((h,), (one, torch.zeros_like(end)))):
        alone = torch.autograd.grad(outs[0] if outs[0] is end else outs[0].sum(), (x, g, s), dend if outs[0] is end else None, retain_graph=True)
        both_given = torch.autograd.grad((h, end), (x, g, s), full, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(alone, both_given))


@pytest.mark.gpu
def test_a_second_derivative_raises():
    x = torch.randn(1, 20, 8, device="cuda").requires_grad_()
    h, _ = kla_b200.gated_scan_b200(x, x * 2)
    dx, = torch.autograd.grad(h.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.gpu
def test_only_the_gradients_that_are_wanted():
    both, h0, dh, _ = (t.cuda() for t in inputs(2, 90, 64, 2, torch.float32))
    x, g = both[..., :64], both[..., 64:]
    full = None
    for wanted in ((0, 1, 2), (0,), (1,), (2,)):
        args = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((x, g, h0))]
        h, end = kla_b200.gated_scan_b200(*args)
        got = dict(zip(wanted, torch.autograd.grad(h, [args[i] for i in wanted], dh)))
        full = full or got
        assert all(torch.equal(got[i], full[i]) for i in wanted)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,D", [(1, 1), (3, 65), (32, 2048)])
def test_tokens_continue_a_prompt(B, D, dtype):
    both, h0, _, _ = inputs(B, 40, D, B, dtype)
    both, state = both.cuda(), h0.cuda()
    x, g = both[..., :D], both[..., D:]
    want, err = oracle(*(t.double().cpu().numpy() for t in (x, g, h0)))
    _, state = kla_b200.gated_scan_b200(x[:, :30], g[:, :30], state)
    kept = state.clone()
    for t in range(30, 40):
        h, new = kla_b200.gated_step_b200(x[:, t], g[:, t], state)
        assert torch.equal(state, kept)
        h2, same = kla_b200.gated_step_b200(x[:, t], g[:, t], state, state_out=state)
        assert same is state or same.data_ptr() == state.data_ptr()
        assert torch.equal(h, h2) and torch.equal(state, new)
        held(h, want["h"][:, t], err["h"][:, t], f"token {t}")
        kept = state.clone()
    held(state, want["end"], err["end"], "state")


@pytest.mark.gpu
def test_captured_and_on_another_stream():
    both, h0, dh, dend = (t.cuda() for t in inputs(2, 333, 96, 2, torch.bfloat16))
    x, g, s = (t.detach().requires_grad_() for t in (both[..., :96], both[..., 96:], h0))

    def step():
        h, end = kla_b200.gated_scan_b200(x, g, s)
        return (h.detach(), end.detach(), *torch.autograd.grad((h, end), (x, g, s), (dh, dend)))

    want = [t.clone() for t in step()]
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
        for t in got:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():  # new values in the same places
        both.copy_(both.flip(1))
    again = [t.clone() for t in step()]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, again)) and not torch.equal(again[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_waits_that_run_out_are_reported_and_the_next_call_is_right(dtype):
    """One sequence of few channels is shared by a cluster of CTAs, which wait for one another's maps."""
    L = lib.load()
    both, _, dh, _ = (t.cuda() for t in inputs(1, 2000, 64, 1, dtype))
    x, g = (t.requires_grad_() for t in (both[..., :64], both[..., 64:]))

    def step():
        h, _ = kla_b200.gated_scan_b200(x, g)
        return h, lambda: torch.autograd.grad(h, (x, g), dh, retain_graph=True)

    h0, grads0 = step()
    grads0 = grads0()
    assert lib.device_status() == 0
    for where in ("forward", "backward"):
        h, grads = step()
        try:
            assert L.kla_b200_test_hooks(3_000_000, 1) == 0  # 3 ms; the second round's maps are not sent
            step() if where == "forward" else grads()
            st = lib.device_status()
        finally:
            assert L.kla_b200_test_hooks(0, -1) == 0
        assert st == 0x150, hex(st)
        h, grads = step()
        assert torch.equal(h, h0) and all(torch.equal(a, b) for a, b in zip(grads(), grads0)) and lib.device_status() == 0


def gated_refusals(dev):
    x = torch.zeros(2, 3, 4, device=dev)
    s = torch.zeros(2, 4, device=dev)
    cu = torch.zeros(3, dtype=torch.int32, device=dev)
    scan, step = kla_b200.gated_scan_b200, kla_b200.gated_step_b200
    return [
        (ValueError, lambda: scan(x, x[:, :2])),
        (ValueError, lambda: scan(x[0], x[0])),
        (ValueError, lambda: scan(x, x.bfloat16())),
        (NotImplementedError, lambda: scan(x.double(), x.double())),
        (NotImplementedError, lambda: scan(x.half(), x.half())),
        (ValueError, lambda: scan(x, x, s[:1])),
        (ValueError, lambda: scan(x, x, s.double())),
        (ValueError, lambda: scan(x, x, s.cpu())),
        (ValueError, lambda: scan(x, x, cu_seqlens=cu)),
        (ValueError, lambda: scan(x[:1], x[:1], cu_seqlens=cu.float())),
        (ValueError, lambda: scan(x[:1], x[:1], cu_seqlens=cu.cpu())),
        (ValueError, lambda: scan(x[:1], x[:1], cu_seqlens=cu[:0])),
        (ValueError, lambda: scan(x[:1], x[:1], s[:1], cu_seqlens=cu)),
        (ValueError, lambda: step(x, x, s)),
        (ValueError, lambda: step(x[:, 0], x[:, 0], s[:1])),
        (ValueError, lambda: step(x[:, 0], x[:, 0], s, s.bfloat16())),
        (ValueError, lambda: step(x[:, 0], x[:, 0], s, torch.zeros(4, 2, device=dev).t())),
        (NotImplementedError, lambda: step(x[:, 0].clone().requires_grad_(), x[:, 0], s)),
        (RuntimeError, lambda: (lambda buf: step(x[:, 0], x[:, 0], buf[:2], buf[1:]))(torch.zeros(3, 4, device=dev))),
    ]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(19))
def test_refusals(i):
    error, call = gated_refusals("cuda")[i]
    with pytest.raises(error):
        call()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 4)
    with pytest.raises(NotImplementedError):
        kla_b200.gated_scan_b200(x, x)
    with pytest.raises(NotImplementedError):
        kla_b200.gated_scan_b200(x.requires_grad_(), x)
    with pytest.raises(NotImplementedError):
        kla_b200.gated_step_b200(x[:, 0], x[:, 0], x[:, 0])


def test_entry_points_reject_bad_arguments_without_cuda():
    L = lib.load()
    A = lambda **kw: ctypes.byref(lib.GatedArgs(**{**dict(B=2, L=4, D=8, sequences=2, dtype=0), **kw}))  # noqa: E731
    T = lambda p: lib.Tensor3(ptr=p, stride_b=32, stride_t=8)  # noqa: E731
    full = dict(x=T(64), gate=T(64), h=T(64), state_out=64, ckpt=64, dh=T(64), dx=T(64), dgate=T(64))
    for fn in (L.kla_b200_gated_scan_fwd, L.kla_b200_gated_scan_bwd):
        assert fn(None, None) == 1
        assert fn(A(), None) == 1                                        # NULL tensors
        assert fn(A(**full, B=-1), None) == 1
        assert fn(A(**full, dtype=5), None) == 2
        assert fn(A(**full, L=1 << 31), None) == 2
        assert fn(A(**full, sequences=3), None) == 1                     # not the batch entries
        assert fn(A(**full, cu_seqlens=64), None) == 1                   # packed sequences of two batch entries
        assert fn(A(**{**full, "x": T(66)}), None) == 4
        assert fn(A(**full, state=66), None) == 4
        assert fn(A(**full, D=0), None) == 0
        assert fn(A(**full, B=0, sequences=0), None) == 0
    assert L.kla_b200_gated_scan_fwd(A(**{**full, "state_out": None}), None) == 1
    assert L.kla_b200_gated_scan_bwd(A(**{**full, "ckpt": None}), None) == 1
    S = lambda **kw: ctypes.byref(lib.GatedStepArgs(**{**dict(B=2, D=8, x=64, gate=64, state=64, state_out=64, h=64), **kw}))  # noqa: E731
    assert L.kla_b200_gated_step(None, None) == 1
    assert L.kla_b200_gated_step(S(x=None), None) == 1
    assert L.kla_b200_gated_step(S(dtype=3), None) == 2
    assert L.kla_b200_gated_step(S(h=66), None) == 4
    assert L.kla_b200_gated_step(S(B=0), None) == 0
    size = L.kla_b200_gated_ckpt_bytes
    assert size(3, 65, 10, 0) == 3 * 2 * 10 * 4 and size(3, 65, 10, 1) == (1 + 3 + 1) * 10 * 4
    assert size(0, 5, 5, 0) == 0 and size(1 << 30, 1 << 30, 1 << 30, 0) == 2 ** 64 - 1


def test_units_of_packed_sequences_do_not_meet():
    """The forward's states lie at lo // 64 + n + step // 64: apart for all sequences, and within the scratch."""
    rng = np.random.default_rng(0)
    for _ in range(200):
        L, n = int(rng.integers(0, 700)), int(rng.integers(1, 9))
        cuts = np.sort(np.concatenate(([0, L], rng.integers(0, L + 1, n - 1))))
        used = [lo // 64 + i + u for i, (lo, hi) in enumerate(zip(cuts[:-1], cuts[1:])) for u in range(-(-(hi - lo) // 64))]
        assert len(set(used)) == len(used)
        assert all(4 * (u + 1) <= lib.load().kla_b200_gated_ckpt_bytes(n, L, 1, 1) for u in used)
