"""The gated recurrence and the gated feed-forward block together, as the two halves of a recurrent block: trained over a batch of
sequences, and decoded token by token from a prompt's state. Held to what torch's own bfloat16 operations make of the same
block: both are compared with float64, and the kernels' error may be 1.5 times that of torch's operations (they round in fewer
places, but sum in another order)."""

import pytest
import torch
import torch.nn.functional as F

import kla_b200

pytestmark = pytest.mark.gpu


def weights(d, M, H, seed=0):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).bfloat16().cuda()  # noqa: E731
    bias = torch.cat((torch.zeros(M), torch.full((M,), 2.0))).bfloat16().cuda()  # gates that hold
    return dict(w_in=rn(2 * M, d), b_in=bias, w_out=rn(d, M), w12=rn(2 * H, d), w3=rn(d, H))


def block(x, state, w, scan, mlp):
    p = F.linear(x, w["w_in"], w["b_in"])
    h, state = scan(*p.chunk(2, -1), state)
    y = x + F.linear(h.to(x.dtype), w["w_out"])
    return mlp(y, w), state


def scan_by_steps(x, gate, state):
    """Step by step, in float32 at least."""
    T = torch.promote_types(x.dtype, torch.float32)
    a, h, out = torch.sigmoid(gate.to(T)), state.to(T), []
    for t in range(x.shape[1]):
        h = a[:, t] * h + torch.sigmoid(-gate[:, t].to(T)) * x[:, t].to(T)
        out.append(h)
    return torch.stack(out, 1), h


def mlp_by_operations(y, w):
    g, u = F.linear(y, w["w12"]).chunk(2, -1)
    return y + F.linear(F.silu(g) * u, w["w3"])


def own(x, state, w):
    return block(x, state, w, kla_b200.gated_scan_b200, lambda y, w: kla_b200.gated_mlp_b200(y, w["w12"], w["w3"], residual=y))


def off(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("B,L,d,M,H", [(2, 300, 64, 96, 168), (1, 1100, 128, 128, 344), (9, 33, 72, 40, 56)])
def test_training(B, L, d, M, H):
    g = torch.Generator().manual_seed(1)
    x, state, dy = torch.randn(B, L, d, generator=g).bfloat16().cuda(), torch.randn(B, M, generator=g).cuda(), torch.randn(B, L, d, generator=g).bfloat16().cuda()
    w = weights(d, M, H)

    def run(f, T):
        leaves = [t.to(T if t.dtype == torch.bfloat16 else torch.promote_types(T, torch.float32)).detach().requires_grad_() for t in (x, state, *w.values())]
        y, end = f(leaves[0], leaves[1], dict(zip(w, leaves[2:])))
        return [y, end, *torch.autograd.grad((y, end), leaves, (dy.to(T), torch.ones_like(end)))]

    plain = lambda x, s, w: block(x, s, w, scan_by_steps, mlp_by_operations)  # noqa: E731
    exact, torchs, ours = run(plain, torch.float64), run(plain, torch.bfloat16), run(own, torch.bfloat16)
    for name, e, t, o in zip(("y", "state", "dx", "dstate", *("d" + n for n in w)), exact, torchs, ours):
        assert o.dtype == t.dtype and off(o, e) <= 1.5 * off(t, e) + 1e-6, (name, off(o, e), off(t, e))


@pytest.mark.parametrize("B", [1, 8, 40])
def test_tokens_behind_a_prompt(B):
    """The prompt's and the tokens' kernels give one sequence."""
    d, M, H, L, n = 128, 192, 344, 50, 12
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(B, L + n, d, generator=g).bfloat16().cuda(), weights(d, M, H)
    zero = torch.zeros(B, M, device="cuda")
    with torch.no_grad():
        exact, _ = block(x.double(), zero.double(), {k: v.double() for k, v in w.items()}, scan_by_steps, mlp_by_operations)
        torchs, _ = block(x, zero, w, scan_by_steps, mlp_by_operations)
        y, state = own(x[:, :L], zero, w)
        out = [y]
        for t in range(L, L + n):
            p = F.linear(x[:, t], w["w_in"], w["b_in"])
            h, _ = kla_b200.gated_step_b200(*p.chunk(2, -1), state, state_out=state)
            r = x[:, t] + F.linear(h, w["w_out"])
            out.append(kla_b200.gated_mlp_b200(r, w["w12"], w["w3"], residual=r)[:, None])
    for part in (slice(0, L), slice(L, L + n)):
        assert off(torch.cat(out, 1)[:, part], exact[:, part]) <= 1.5 * off(torchs[:, part], exact[:, part]) + 1e-6


def test_two_calls_at_once():
    """Both operators on two streams, forward and backward, do not share working memory."""
    x = [torch.randn(4, 700, 256, device="cuda").bfloat16() for _ in range(2)]
    w, zero = weights(256, 256, 688), torch.zeros(4, 256, device="cuda")

    def step(x):
        leaves = [t.detach().requires_grad_() for t in (x, *w.values())]
        y, _ = own(leaves[0], zero, dict(zip(w, leaves[1:])))
        return torch.autograd.grad(y.sum(), leaves)

    want = [step(t) for t in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s, t in zip(streams, x):
            with torch.cuda.stream(s):
                got.append(step(t))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q))


def test_a_models_prompt_with_the_fused_mlp():
    from test_model_decode_gpu import decoder, model_weights, restated

    layers, w = 3, model_weights(128, 3, 512)
    ids = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(3)).cuda()
    exact = restated(w, layers, ids, torch.float64, torch.float64)
    dec = decoder(w, layers)
    plain, _ = dec.prefill(ids)
    before = dec.generate(ids, 4)
    dec.fused_mlp = True
    fused, state = dec.prefill(ids)
    assert not torch.equal(fused, plain)  # it is another way
    assert off(fused, exact) <= 1.5 * off(plain, exact)
    assert dec.generate(ids, 4).shape == before.shape
    dec.fused_mlp = False
    assert torch.equal(dec.prefill(ids)[0], plain) and torch.equal(dec.generate(ids, 4), before)
