"""The gated recurrence and the gated feed-forward block, as timeable cases.

Two operators that stand next to each other in a recurrent block:

* the gated recurrence ``h_t = a_t h_{t-1} + (1 - a_t) x_t`` with ``a_t = sigmoid(g_t)``, channel by channel, over a batch of
  sequences, over packed sequences of different lengths, and for one token; forward and backward;
* the gated feed-forward block ``y = (act(x Wg^T + bg) * (x Wu^T + bu)) W3^T + b3 (+ residual)``, forward and backward.

``listed()`` names the cases, ``draw`` gives more of the same ranges, ``prepare`` makes a case's inputs on the GPU and ``run`` is
one pass: elementary torch operations in 32 bits where ``own`` is false, the package's operators where it is true. ``exact`` gives
the same outputs in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of one layer's recurrence at serving batch: latency only
        dict(name="scan_step", kind="scan_step", B=32, D=2048, dtype="bf16"),
        # a prompt of one sequence, whatever length it has, in float32
        dict(name="scan_one_sequence", kind="scan", B=1, L=1501, D=1536, dtype="f32", carry=False),
        # long prompts of a batch, continued from a state and leaving one for the tokens that follow
        dict(name="scan_prompts", kind="scan", B=4, L=8192, D=2048, dtype="bf16", carry=True),
        # a training step of a layer's recurrence: 16 sequences of 2048 in bfloat16
        dict(name="scan_train", kind="scan_train", B=16, L=2048, D=1536, dtype="bf16", carry=False, packed=0),
        # training on packed sequences of different lengths, some empty, sizes that divide into nothing
        dict(name="scan_train_packed", kind="scan_train", B=1, L=6001, D=1001, dtype="f32", carry=True, packed=9),
        # training on one long context from a carried state
        dict(name="scan_train_long", kind="scan_train", B=1, L=65536, D=4096, dtype="bf16", carry=True, packed=0),
        # one token of eight sequences through the block: latency, the weights' read
        dict(name="mlp_token", kind="mlp", rows=8, d=768, H=2048, act="silu", bias=False, residual=True),
        # the prompts of eight sequences of 512
        dict(name="mlp_prompts", kind="mlp", rows=4096, d=768, H=2048, act="silu", bias=False, residual=True),
        # training with biases at a width of 8/3 d_model that was not rounded
        dict(name="mlp_train_ragged", kind="mlp_train", rows=1501, d=512, H=1365, act="silu", bias=True, residual=False),
        # a training step of the 768-wide block: 16 sequences of 2048
        dict(name="mlp_train", kind="mlp_train", rows=32768, d=768, H=2048, act="silu", bias=False, residual=False),
        # a training step of a wide block
        dict(name="mlp_train_wide", kind="mlp_train", rows=8192, d=2048, H=5456, act="silu", bias=False, residual=True),
    ]


def _log(rng, lo, hi):
    """A size between ``lo`` and ``hi``, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def _width(rng, lo, hi, step):
    """A width: mostly a multiple of ``step`` as layers have it, sometimes any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(step, n // step * step)


def draw(rng):
    kind = rng.choice(["scan_step", "scan", "scan_train", "scan_train", "mlp", "mlp", "mlp_train", "mlp_train"])
    if kind == "scan_step":
        return dict(kind=kind, B=_log(rng, 1, 256), D=_width(rng, 64, 4096, 64), dtype=rng.choice(["f32", "bf16"]))
    if kind in ("scan", "scan_train"):
        B, D = _log(rng, 1, 16), _width(rng, 64, 4096, 64)
        case = dict(kind=kind, B=B, L=_log(rng, 1, min(65536, 2 ** 27 // (B * D))), D=D, dtype=rng.choice(["f32", "bf16"]),
                    carry=rng.random() < 0.5)
        if kind == "scan_train":
            case["packed"] = 0
            if rng.random() < 0.3:
                case.update(B=1, L=B * case["L"], packed=_log(rng, 1, 64))
        return case
    d = _width(rng, 64, 2048, 64)
    H = _width(rng, 2 * d, 4 * d, 8)
    most = 8192 * 2048 * 5456 // (d * H)
    rows = _log(rng, 1, min(32768, most)) if kind == "mlp" else _log(rng, 64, min(32768, most))
    return dict(kind=kind, rows=rows, d=d, H=H, act=rng.choice(["silu", "silu", "silu", "gelu", "relu"]), bias=rng.random() < 0.4,
                residual=rng.random() < 0.5)


# --- inputs ------------------------------------------------------------------------------------------------------


def _random(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return g, lambda *shape, scale=1.0: torch.randn(*shape, generator=g, device="cuda").mul_(scale)


def _bounds(total, n, seed):
    """Bounds of ``n`` sequences that fill ``total`` rows: lengths of any size, some of them zero."""
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, total + 1, (n - 1,), generator=g).sort().values
    if n > 3:
        cuts[1] = cuts[0]  # an empty sequence
    return torch.cat((torch.zeros(1, dtype=torch.long), cuts, torch.full((1,), total))).to(device="cuda", dtype=torch.int32)


def prepare(case, seed):
    g, rn = _random(seed)
    if case["kind"].startswith("scan"):
        T, D = DTYPES[case["dtype"]], case["D"]
        if case["kind"] == "scan_step":
            B = case["B"]
            both = rn(B, 2 * D).to(T)  # what the layer's projection wrote: input and gate side by side
            both[:, D:] += 2.0  # gates that keep most of the state
            return dict(case, x=both[:, :D], gate=both[:, D:], state=rn(B, D))
        B, L, n = case["B"], case["L"], case.get("packed") or case["B"]
        both = rn(B, L, 2 * D).to(T)
        both[..., D:] += 2.0
        st = dict(case, x=both[..., :D], gate=both[..., D:], state=rn(n, D) if case["carry"] else None,
                  bounds=_bounds(L, n, seed) if case.get("packed") else None)
        if case["kind"] == "scan_train":
            st.update(x=st["x"].requires_grad_(), gate=st["gate"].requires_grad_(), dh=rn(B, L, D).to(T), dstate=rn(n, D))
            if case["carry"]:
                st["state"].requires_grad_()
        return st
    rows, d, H = case["rows"], case["d"], case["H"]
    b = torch.bfloat16
    st = dict(case, x=rn(rows, d).to(b), w12=rn(2 * H, d, scale=d ** -0.5).to(b), w3=rn(d, H, scale=H ** -0.5).to(b),
              b12=rn(2 * H, scale=0.1).to(b) if case["bias"] else None, b3=rn(d, scale=0.1).to(b) if case["bias"] else None,
              residual=rn(rows, d).to(b) if case["residual"] else None)
    if case["kind"] == "mlp_train":
        for name in ("x", "w12", "w3", "b12", "b3"):
            if st[name] is not None:
                st[name].requires_grad_()
        st["dy"] = rn(rows, d).to(b)
    return st


# --- the operators in elementary operations ----------------------------------------------------------------------


def _scan(a, b):
    """``h_t = a_t h_{t-1} + b_t`` along dim 1 from zero: maps of stretches, composed with those of twice the length each round."""
    step = 1
    while step < a.shape[1]:
        h = b.clone()
        h[:, step:] += a[:, step:] * b[:, :-step]
        p = a.clone()
        p[:, step:] *= a[:, :-step]
        a, b, step = p, h, 2 * step
    return b


def _edges(st):
    """Batch index, first and last row of every sequence, and whether it has rows at all (packed sequences: of the one batch)."""
    B, L = st["x"].shape[:2]
    if st["bounds"] is None:
        i = torch.arange(B, device="cuda")
        return i, torch.zeros_like(i), torch.full_like(i, L - 1), torch.ones_like(i, dtype=torch.bool)
    lo, hi = st["bounds"][:-1].long(), st["bounds"][1:].long()
    return torch.zeros_like(lo), lo.clamp_max(L - 1), (hi - 1).clamp_min(0), hi > lo


def _plain_scan(st):
    x, z = st["x"].detach().float(), torch.sigmoid(-st["gate"].detach().float())
    a, (n, D) = 1 - z, (st["B"] if st["bounds"] is None else st["packed"], st["D"])
    state = torch.zeros(n, D, device="cuda") if st["state"] is None else st["state"].detach()
    batch, first, last, some = _edges(st)
    keep, inc = a.clone(), z * x
    # a sequence's first step takes the state it starts from and nothing of the row before (empty ones share a row: add nothing)
    inc.index_put_((batch, first), torch.where(some[:, None], a[batch, first] * state, 0.0), accumulate=True)
    keep[batch[some], first[some]] = 0.0
    h = _scan(keep, inc)
    end = torch.where(some[:, None], h[batch, last], state)
    out = [h.to(st["x"].dtype), end]
    if st["kind"] == "scan":
        return out
    # c_t = dh_t + a_{t+1} c_{t+1}, from the end of every sequence
    dh = st["dh"].float().index_put((batch, last), torch.where(some[:, None], st["dstate"], 0.0), accumulate=True)
    nxt = torch.zeros_like(a)
    nxt[:, :-1] = keep[:, 1:]
    c = _scan(nxt.flip(1), dh.flip(1)).flip(1)
    before = torch.zeros_like(h)
    before[:, 1:] = h[:, :-1]
    before[batch[some], first[some]] = state[some]
    out += [(z * c).to(st["x"].dtype), (c * (before - x) * z * a).to(st["x"].dtype)]
    if st["state"] is not None:
        out.append(torch.where(some[:, None], a[batch, first] * c[batch, first], st["dstate"]))
    return out


def _plain_step(st):
    x, z = st["x"].float(), torch.sigmoid(-st["gate"].float())
    h = (1 - z) * st["state"] + z * x
    return [h.to(st["x"].dtype), h]


def _act(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    return g.clamp_min(0.0), (g > 0).to(g.dtype)


def _plain_mlp(st):
    T, H = st["x"].dtype, st["H"]
    x, w12, w3 = (st[n].detach().float() for n in ("x", "w12", "w3"))
    gu = x @ w12.t()
    if st["bias"]:
        gu = gu + st["b12"].detach().float()
    g, u = gu[:, :H], gu[:, H:]
    f, df = _act(g, st["act"])
    h = f * u
    y = h @ w3.t()
    if st["bias"]:
        y = y + st["b3"].detach().float()
    if st["residual"] is not None:
        y = y + st["residual"].float()
    if st["kind"] == "mlp":
        return [y.to(T)]
    dy = st["dy"].float()
    dh = dy @ w3
    dgu = torch.cat((dh * u * df, dh * f), dim=1)
    out = [y, dgu @ w12, dgu.t() @ x, dy.t() @ h]
    if st["bias"]:
        out += [dgu.sum(0), dy.sum(0)]
    return [t.to(T) for t in out]


def run(state):
    st = state
    if not own:
        if st["kind"] == "scan_step":
            return _plain_step(st)
        return _plain_scan(st) if st["kind"].startswith("scan") else _plain_mlp(st)
    import kla_b200

    if st["kind"] == "scan_step":
        return list(kla_b200.gated_step_b200(st["x"], st["gate"], st["state"]))
    if st["kind"] == "scan":
        with torch.no_grad():
            return list(kla_b200.gated_scan_b200(st["x"], st["gate"], st["state"], cu_seqlens=st["bounds"]))
    if st["kind"] == "scan_train":
        leaves = [st[n] for n in ("x", "gate", "state") if st[n] is not None]
        h, end = kla_b200.gated_scan_b200(st["x"], st["gate"], st["state"], cu_seqlens=st["bounds"])
        return [h.detach(), end.detach(), *torch.autograd.grad((h, end), leaves, (st["dh"], st["dstate"]))]
    given = dict(b12=st["b12"], b3=st["b3"], residual=st["residual"], activation=st["act"])
    if st["kind"] == "mlp":
        with torch.no_grad():
            return [kla_b200.gated_mlp_b200(st["x"], st["w12"], st["w3"], **given)]
    y = kla_b200.gated_mlp_b200(st["x"], st["w12"], st["w3"], **given)
    leaves = [st[n] for n in ("x", "w12", "w3", "b12", "b3") if st[n] is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, st["dy"])]


# --- the work of a pass, and its outputs in 64 bits --------------------------------------------------------------


def work(case):
    if case["kind"].startswith("scan"):
        e, D = (2 if case["dtype"] == "bf16" else 4), case["D"]
        if case["kind"] == "scan_step":
            n = case["B"] * D
            return dict(bytes=3 * e * n + 8 * n, flops=8 * n)
        n = case["B"] * case["L"] * D
        states = 4 * D * (case.get("packed") or case["B"])
        if case["kind"] == "scan":  # x, gate in, h and the state out
            return dict(bytes=3 * e * n + states * (1 + case["carry"]), flops=8 * n)
        return dict(bytes=6 * e * n + states * (2 + 2 * case["carry"]), flops=22 * n)  # also dh in, dx and dgate out
    rows, d, H = case["rows"], case["d"], case["H"]
    weights, acts, biases = 3 * d * H, rows * d, (2 * H + d) * case["bias"]
    if case["kind"] == "mlp":
        return dict(bytes=2 * (weights + biases + (2 + case["residual"]) * acts), flops=6 * rows * d * H)
    return dict(bytes=2 * (2 * weights + 2 * biases + (4 + case["residual"]) * acts), flops=18 * rows * d * H)


def _exact_scan(st):
    """Sequences side by side in 64 bits: a step at a time within stretches, then stretch after stretch."""
    rows, D = st["B"] * st["L"], st["D"]
    flat = lambda t: t.detach().double().reshape(rows, D)  # noqa: E731
    x, e = flat(st["x"]), torch.exp(-flat(st["gate"]))
    a, z = 1 / (1 + e), e / (1 + e)
    if st["bounds"] is None:
        lo = torch.arange(st["B"], device="cuda") * st["L"]
        hi = lo + st["L"]
    else:
        lo, hi = st["bounds"][:-1].long(), st["bounds"][1:].long()
    start = torch.zeros(len(lo), D, device="cuda", dtype=torch.float64) if st["state"] is None else st["state"].detach().double()
    full = (hi > lo).nonzero().squeeze(1)
    lo, hi = lo[full], hi[full]

    def recur(a, b):
        size = max(1, math.isqrt(rows))
        pad = -rows % size
        a = torch.cat((a, a.new_ones(pad, D))).reshape(-1, size, D)
        b = torch.cat((b, b.new_zeros(pad, D))).reshape(-1, size, D)
        h, p = b.clone(), a.clone()
        for t in range(1, size):
            h[:, t] += a[:, t] * h[:, t - 1]
            p[:, t] *= p[:, t - 1]
        carry = torch.zeros_like(h[:, 0])
        for i in range(1, h.shape[0]):
            carry[i] = h[i - 1, -1] + p[i - 1, -1] * carry[i - 1]
        return (h + p * carry[:, None]).reshape(-1, D)[:rows]

    b = z * x
    b[lo] += a[lo] * start[full]
    link = a.clone()
    link[lo] = 0.0
    h = recur(link, b)
    end = start.clone()
    end[full] = h[hi - 1]
    shape = st["x"].shape
    out = [h.reshape(shape), end]
    if st["kind"] == "scan":
        return out
    c = flat(st["dh"]).clone()
    c[hi - 1] += st["dstate"].double()[full]
    c = recur(torch.cat((link[1:], torch.zeros_like(link[:1]))).flip(0), c.flip(0)).flip(0)
    before = torch.cat((torch.zeros_like(h[:1]), h[:-1]))
    before[lo] = start[full]
    out += [(z * c).reshape(shape), (a * z * c * (before - x)).reshape(shape)]
    if st["state"] is not None:
        dstart = st["dstate"].double()
        dstart[full] = a[lo] * c[lo]
        out.append(dstart)
    return out


def _exact_mlp(st):
    """By automatic differentiation in 64 bits."""
    leaves = {n: st[n].detach().double().requires_grad_(st["kind"] == "mlp_train") for n in ("x", "w12", "w3", "b12", "b3") if st[n] is not None}
    gate, up = (torch.nn.functional.linear(leaves["x"], w, b) for w, b in zip(
        leaves["w12"].chunk(2), leaves["b12"].chunk(2) if st["bias"] else (None, None)))
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.nn.functional.relu}[st["act"]]
    y = torch.nn.functional.linear(act(gate) * up, leaves["w3"], leaves.get("b3"))
    if st["residual"] is not None:
        y = y + st["residual"].double()
    if st["kind"] == "mlp":
        return [y]
    return [y.detach(), *torch.autograd.grad(y, list(leaves.values()), st["dy"].double())]


def exact(case, seed):
    if work(case)["flops"] > 3e14 or (case["kind"].startswith("scan") and case["kind"] != "scan_step" and case["B"] * case["L"] * case["D"] > 3e8):
        return None  # over 20 seconds, or over the card's memory
    st = prepare(case, seed)
    if case["kind"] == "scan_step":
        a = torch.sigmoid(st["gate"].double())
        h = a * st["state"].double() + torch.sigmoid(-st["gate"].double()) * st["x"].double()
        return [h, h]
    with torch.enable_grad():
        return _exact_scan(st) if case["kind"].startswith("scan") else _exact_mlp(st)
