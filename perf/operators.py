"""The encoder operators' measured cases: the gated linear recurrence, the gated
residual norm and the 8-bit activation checkpoints, each in a plain form
(elementary torch operations in 32 bits) and through this package's kernels.

``own`` chooses which of the two ``run`` computes.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 32  # channels of a token that share a scale in the 8-bit checkpoints
EPS = 1e-6

# the largest listed recurrence, norm and weight gradient: what a drawn case may cost at most
MOST_SCAN = 64 * 10000 * 512
MOST_NORM = 32 * 4096 * 512
MOST_PACK = 1000000 * 512
MOST_PRODUCT = 32 * 4096 * 512 * 1536


def listed():
    return [
        # serving: one token of a few streams, where latency counts, and of a full batch
        dict(name="step_few", op="step", dtype="bf16", B=4, D=512),
        dict(name="step_batch", op="step", dtype="fp32", B=512, D=1024),
        # inference over one chromosome: a single sequence of a million positions
        dict(name="scan_chromosome", op="scan", dtype="bf16", B=1, T=1000000, D=512, train=False,
             reverse=False, ragged=False),
        # training at the framework's default workload (batch 64, 10^4 positions), ragged lengths
        dict(name="scan_train", op="scan", dtype="bf16", B=64, T=10000, D=512, train=True,
             reverse=False, ragged=True),
        # the quick-start's shape (batch 4, 1000 positions, hidden 512), the backward direction of a
        # bidirectional encoder, 32 bits
        dict(name="scan_train_small", op="scan", dtype="fp32", B=4, T=1000, D=512, train=True,
             reverse=True, ragged=True),
        # odd width and length, 16-bit floats
        dict(name="scan_train_odd", op="scan", dtype="fp16", B=3, T=4097, D=203, train=True,
             reverse=False, ragged=True),
        # inference through the norms of one block at the quick-start's shape
        dict(name="norm_small", op="norm", dtype="bf16", B=4, T=1000, D=512, train=False,
             ragged=False),
        # a training step through them: batch 32, 4096 positions
        dict(name="norm_train", op="norm", dtype="bf16", B=32, T=4096, D=512, train=True,
             ragged=False),
        # odd width, ragged, 32 bits
        dict(name="norm_train_odd", op="norm", dtype="fp32", B=5, T=1777, D=203, train=True,
             ragged=True),
        # the checkpoint of a long activation, stored and read back
        dict(name="pack_long", op="pack", dtype="bf16", B=1, T=1000000, D=512, ragged=False),
        # the gradient of an in-projection's weight (512 -> 3 * 512) from its stored input
        dict(name="weight_grad", op="weight_grad", dtype="bf16", B=32, T=4096, D=512, M=1536,
             ragged=False),
        # odd widths, ragged, 32 bits
        dict(name="weight_grad_odd", op="weight_grad", dtype="fp32", B=4, T=1000, D=203, M=509,
             ragged=True),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm; odd sizes and round ones alike."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.4 and n >= 16:
        n -= n % (8 if n < 256 else 64)
    return max(lo, min(hi, n))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "norm", "norm", "pack", "weight_grad"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    width = 1 if dtype != "fp32" else 2  # a 32-bit case costs twice a 16-bit one
    if op == "step":
        return dict(op=op, dtype=dtype, B=_log_int(rng, 1, 512), D=_log_int(rng, 64, 1024))
    B, D = _log_int(rng, 1, 64), _log_int(rng, 32, 1024)
    ragged = rng.random() < 0.5
    if op == "scan":
        T = _log_int(rng, 1, max(1, min(1000000, MOST_SCAN // (B * D * width))))
        return dict(op=op, dtype=dtype, B=B, T=T, D=D, train=rng.random() < 0.7,
                    reverse=rng.random() < 0.5, ragged=ragged)
    if op == "norm":
        T = _log_int(rng, 1, max(1, MOST_NORM // (B * D * width)))
        return dict(op=op, dtype=dtype, B=B, T=T, D=D, train=rng.random() < 0.7, ragged=ragged)
    if op == "pack":
        T = _log_int(rng, 1, max(1, MOST_PACK // (B * D * width)))
        return dict(op=op, dtype=dtype, B=B, T=T, D=D, ragged=ragged)
    M = _log_int(rng, 32, 2048)
    T = _log_int(rng, 1, max(1, min(131072 // B, MOST_PRODUCT // (B * D * M * width))))
    return dict(op=op, dtype=dtype, B=B, T=T, D=D, M=M, ragged=ragged)


def _lengths(case, seed):
    """Half to full length, among larger batches one empty sequence and one of one position."""
    g = torch.Generator().manual_seed(seed + 77)
    B, T = case["B"], case["T"]
    n = torch.randint((T + 1) // 2, T + 1, (B,), generator=g)
    if B >= 3:
        n[B - 1] = 0
        n[B - 2] = 1
    return n


def prepare(case, seed):
    dev = torch.device("cuda")
    dt = DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    B, D = case["B"], case["D"]

    def normal(*shape, scale=1.0, shift=None, dtype=dt):
        v = torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)
        v.mul_(scale)
        if shift is not None:
            v.add_(shift)
        return v.to(dtype)

    # forget gates whose memory reaches from one position to some hundreds, by channel
    bias = torch.linspace(-1.0, 6.0, D, device=dev)
    s = {"case": dict(case)}
    if case["op"] == "step":
        s.update(x=normal(B, D), gate=normal(B, D, shift=bias),
                 state=normal(B, D, dtype=torch.float32))
        return s
    T = case["T"]
    s["lengths"] = _lengths(case, seed).to(dev) if case["ragged"] else None
    train = case.get("train", False)
    if case["op"] == "scan":
        s.update(x=normal(B, T, D).requires_grad_(train),
                 gate=normal(B, T, D, shift=bias).requires_grad_(train),
                 initial=normal(B, D, dtype=torch.float32).requires_grad_(train))
        if train:
            s.update(grad_h=normal(B, T, D), grad_state=normal(B, D, dtype=torch.float32))
    elif case["op"] == "norm":
        s.update(residual=normal(B, T, D, scale=2.0).requires_grad_(train),
                 branch=normal(B, T, D, scale=0.5).requires_grad_(train),
                 gate=normal(B, T, D).requires_grad_(train))
        for name, mean in (("branch_weight", 1.0), ("residual_scale", 0.3), ("next_weight", 1.0)):
            s[name] = normal(D, scale=0.1, shift=mean, dtype=torch.float32).requires_grad_(train)
        if train:
            s.update(grad_residual=normal(B, T, D), grad_normed=normal(B, T, D))
    else:
        # a norm's output: unit scale with a few large channels
        spread = torch.ones(D, device=dev)
        spread[:: 37] = 12.0
        x = torch.randn(B, T, D, generator=gen, device=dev, dtype=torch.float32)
        s["x"] = x.mul_(spread).to(dt)
        if case["op"] == "weight_grad":
            s["grad_output"] = normal(B, T, case["M"])
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from h = 0, by doubling the distance
    that each position's (a, b) reaches back: log2(T) elementwise passes."""
    T, step = a.shape[1], 1
    while step < T:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], dim=1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], dim=1)
        step *= 2
    return b


def _valid(s, T):
    """(B, T, 1) truth values of the positions below each length; None where all are."""
    if s["lengths"] is None:
        return None
    return (torch.arange(T, device=s["lengths"].device) < s["lengths"][:, None])[..., None]


def _keep(v, valid):
    return v if valid is None else torch.where(valid, v, torch.zeros_like(v))


def _plain_scan(s):
    case, dt = s["case"], s["x"].dtype
    valid = _valid(s, case["T"])
    x, g = s["x"].float(), s["gate"].float()
    f, i = torch.sigmoid(g), torch.sigmoid(-g)
    if valid is not None:  # a masked position leaves the state as it is
        f = torch.where(valid, f, torch.ones_like(f))
        i = torch.where(valid, i, torch.zeros_like(i))
        x = torch.where(valid, x, torch.zeros_like(x))
    if case["reverse"]:
        x, f, i = x.flip(1), f.flip(1), i.flip(1)
    b = i * x
    b[:, 0] += f[:, 0] * s["initial"]
    h = _scan(f, b)
    state = h[:, -1].clone()
    out = h.flip(1) if case["reverse"] else h
    out = _keep(out, valid).to(dt)
    if not case["train"]:
        return {"h": out, "state": state}
    dh = _keep(s["grad_h"].float(), valid)
    dh = dh.flip(1) if case["reverse"] else dh
    dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["grad_state"][:, None]], dim=1)
    # the same recurrence from the other end, with each position's successor's forget gate
    after = torch.cat([f[:, 1:], torch.zeros_like(f[:, :1])], dim=1)
    lam = _scan(after.flip(1), dh.flip(1)).flip(1)
    before = torch.cat([s["initial"][:, None], h[:, :-1]], dim=1)
    dx, dg = lam * i, lam * (before - x) * f * i
    dinit = lam[:, 0] * f[:, 0]
    if case["reverse"]:
        dx, dg = dx.flip(1), dg.flip(1)
    return {"h": out, "state": state, "grad_x": dx.to(dt), "grad_gate": dg.to(dt),
            "grad_initial": dinit}


def _plain_step(s):
    x, g = s["x"].float(), s["gate"].float()
    h = torch.sigmoid(g) * s["state"] + torch.sigmoid(-g) * x
    return {"h": h.to(s["x"].dtype), "state": h}


def _plain_norm(s):
    case, dt = s["case"], s["residual"].dtype
    D = case["D"]
    valid = _valid(s, case["T"])
    x, z, g = (_keep(s[k].float(), valid) for k in ("residual", "branch", "gate"))
    w1, sc, w2 = s["branch_weight"], s["residual_scale"], s["next_weight"]
    rz = torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS)
    zh = z * rz
    sig = torch.sigmoid(g)
    u = g * sig
    zn = zh * w1
    r = x + sc * u * zn
    rr = torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)
    n = r * rr * w2
    out = {"residual": r.to(dt), "normed": n.to(dt)}
    if not case["train"]:
        return out
    dr, dn = (_keep(s[k].float(), valid) for k in ("grad_residual", "grad_normed"))
    rh = r * rr
    dnw = dn * w2
    d = dr + rr * (dnw - rh * (dnw * rh).sum(-1, keepdim=True) / D)
    dzn = d * sc * u
    dzw = dzn * w1
    dz = rz * (dzw - zh * (dzw * zh).sum(-1, keepdim=True) / D)
    dg = d * sc * zn * sig * (1 + g * (1 - sig))
    out.update(grad_residual=d.to(dt), grad_branch=dz.to(dt), grad_gate=dg.to(dt),
               grad_branch_weight=(dzn * zh).sum((0, 1)), grad_scale=(d * u * zn).sum((0, 1)),
               grad_next_weight=(dn * rh).sum((0, 1)))
    return out


def _stored(x, valid):
    """What the 8-bit checkpoint of x stands for, in 32 bits: for each 32
    channels of a token, multiples of the smallest power of two 2^e with
    max |x| <= 127 * 2^e (e >= -126), and none past the type's largest value."""
    B, T, D = x.shape
    top = torch.finfo(x.dtype).max
    v = _keep(x.float(), valid)
    v = torch.nn.functional.pad(v, (0, -D % GROUP)).view(B, T, -1, GROUP)
    amax = v.abs().amax(-1, keepdim=True)
    m, p = torch.frexp(amax)
    e = (torch.where(m <= 127.0 / 128.0, p - 7, p - 6)).clamp(min=-126)
    q = torch.round(torch.ldexp(v, -e))
    most = torch.floor(torch.ldexp(torch.full_like(amax, top), -e))
    q = torch.minimum(torch.maximum(q, -most), most)
    v = torch.ldexp(q, e)
    return v.view(B, T, -1)[..., :D]


def _plain_pack(s):
    return {"x": _stored(s["x"], _valid(s, s["case"]["T"])).to(s["x"].dtype)}


def _plain_weight_grad(s):
    valid = _valid(s, s["case"]["T"])
    x = _stored(s["x"], valid)
    dy = _keep(s["grad_output"].float(), valid)
    dw = dy.reshape(-1, dy.shape[-1]).t() @ x.reshape(-1, x.shape[-1])
    return {"grad_weight": dw.to(s["x"].dtype)}


# ---------------------------------------------------------------------------
# the package's operators, as a user calls them
# ---------------------------------------------------------------------------
def _own_scan(s):
    import torch_semimarkov_b200 as tsm

    case = s["case"]
    h, state = tsm.gated_linear_recurrence(s["x"], s["gate"], s["initial"], s["lengths"],
                                           reverse=case["reverse"])
    out = {"h": h.detach(), "state": state.detach()}
    if case["train"]:
        gx, gg, gi = torch.autograd.grad((h, state), (s["x"], s["gate"], s["initial"]),
                                         (s["grad_h"], s["grad_state"]))
        out.update(grad_x=gx, grad_gate=gg, grad_initial=gi)
    return out


def _own_step(s):
    import torch_semimarkov_b200 as tsm

    h, state = tsm.gated_linear_recurrence_step(s["x"], s["gate"], s["state"])
    return {"h": h, "state": state}


def _own_norm(s):
    import torch_semimarkov_b200 as tsm

    leaves = tuple(s[k] for k in ("residual", "branch", "gate", "branch_weight", "residual_scale",
                                  "next_weight"))
    r, n = tsm.gated_residual_norm(*leaves, lengths=s["lengths"], eps=EPS)
    out = {"residual": r.detach(), "normed": n.detach()}
    if s["case"]["train"]:
        names = ("grad_residual", "grad_branch", "grad_gate", "grad_branch_weight", "grad_scale",
                 "grad_next_weight")
        out.update(zip(names, torch.autograd.grad((r, n), leaves,
                                                  (s["grad_residual"], s["grad_normed"]))))
    return out


def _own_pack(s):
    import torch_semimarkov_b200 as tsm

    return {"x": tsm.pack_activation(s["x"], s["lengths"]).unpack()}


def _own_weight_grad(s):
    import torch_semimarkov_b200 as tsm

    packed = tsm.pack_activation(s["x"], s["lengths"])
    return {"grad_weight": tsm.packed_weight_grad(s["grad_output"], packed, s["lengths"])}


PLAIN = {"step": _plain_step, "scan": _plain_scan, "norm": _plain_norm, "pack": _plain_pack,
         "weight_grad": _plain_weight_grad}
OWN = {"step": _own_step, "scan": _own_scan, "norm": _own_norm, "pack": _own_pack,
       "weight_grad": _own_weight_grad}


def run(state):
    op = state["case"]["op"]
    if own:
        return OWN[op](state)
    with torch.no_grad():
        return PLAIN[op](state)


def work(case):
    """What a pass cannot do without: each input read once, each output written once."""
    size = DTYPES[case["dtype"]].itemsize
    op, B, D = case["op"], case["B"], case["D"]
    if op == "step":
        return {"bytes": B * D * (3 * size + 8), "flops": 10 * B * D}
    T = case["T"]
    # about three quarters of a ragged batch's positions are read; all are written
    share = 0.75 if case["ragged"] else 1.0
    E = B * T * D
    if op == "scan":
        streams_in, streams_out, flops = (5, 3, 30) if case["train"] else (2, 1, 10)
        return {"bytes": (share * streams_in + streams_out) * E * size + 8 * B * D,
                "flops": share * flops * E}
    if op == "norm":
        streams_in, streams_out, flops = (8, 5, 60) if case["train"] else (3, 2, 20)
        return {"bytes": (share * streams_in + streams_out) * E * size, "flops": share * flops * E}
    codes = B * T * (D + -(-D // GROUP))
    if op == "pack":
        return {"bytes": share * E * size + 2 * codes + E * size, "flops": share * 4 * E}
    M = case["M"]
    return {"bytes": share * (E * size + B * T * M * size) + 2 * codes + M * D * size,
            "flops": share * 2 * E * M}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _walk(a, b, h0):
    """Every h_t = a_t h_{t-1} + b_t in 64 bits.  The time axis is cut into
    about sqrt(T) runs: all runs walk at once from a zero state beside the
    products of their a, then the runs' ends are joined one after another."""
    B, T, D = a.shape
    n = max(1, math.isqrt(T))
    runs = -(-T // n)
    pad = runs * n - T
    a = torch.nn.functional.pad(a, (0, 0, 0, pad), value=1.0).view(B, runs, n, D)
    h = torch.nn.functional.pad(b, (0, 0, 0, pad)).view(B, runs, n, D).clone()
    p = a.clone()
    for t in range(1, n):
        h[:, :, t] += a[:, :, t] * h[:, :, t - 1]
        p[:, :, t] *= p[:, :, t - 1]
    start = torch.empty(B, runs, D, dtype=a.dtype, device=a.device)
    carry = h0
    for r in range(runs):
        start[:, r] = carry
        carry = h[:, r, -1] + p[:, r, -1] * carry
    h += p * start[:, :, None]
    return h.view(B, runs * n, D)[:, :T]


def _exact_scan(s):
    case = s["case"]
    B, T, D = s["x"].shape
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), T, device=s["x"].device)
    t = torch.arange(T, device=s["x"].device)
    live = (t[None] < n[:, None]).unsqueeze(-1)
    order = t.flip(0) if case["reverse"] else t
    f = (1 / (1 + torch.exp(-s["gate"].detach().double())))
    i = (1 / (1 + torch.exp(s["gate"].detach().double())))
    f = f.masked_fill(~live, 1.0)[:, order]
    i = i.masked_fill(~live, 0.0)[:, order]
    x = s["x"].detach().double().masked_fill(~live, 0.0)[:, order]
    h0 = s["initial"].detach().double()
    h = _walk(f, i * x, h0)
    out = {"h": h[:, order].masked_fill(~live, 0.0), "state": h[:, -1].clone()}
    if not case["train"]:
        return out
    dh = s["grad_h"].double().masked_fill(~live, 0.0)[:, order]
    # d loss / d h_t gathers what reaches position t from all later ones
    nxt = torch.ones_like(f)
    nxt[:, :-1] = f[:, 1:]
    lam = _walk(nxt.flip(1), dh.flip(1), s["grad_state"].double()).flip(1)
    del nxt, dh
    prev = torch.empty_like(h)
    prev[:, 1:], prev[:, 0] = h[:, :-1], h0
    out["grad_x"] = (lam * i)[:, order]
    out["grad_gate"] = (lam * (prev - x) * f * i)[:, order]
    out["grad_initial"] = lam[:, 0] * f[:, 0]
    return out


def _exact_norm(s):
    """The forward definition in 64 bits; its gradients by automatic differentiation."""
    case = s["case"]
    names = ("residual", "branch", "gate", "branch_weight", "residual_scale", "next_weight")
    B, T, D = s["residual"].shape
    rows = torch.ones(B, T, dtype=torch.bool, device=s["residual"].device)
    if s["lengths"] is not None:
        rows = torch.arange(T, device=rows.device)[None] < s["lengths"][:, None]
    with torch.set_grad_enabled(case["train"]):
        full = [s[k].detach().double().requires_grad_(case["train"]) for k in names]
        x, z, g = (v[rows] for v in full[:3])
        w1, sc, w2 = full[3:]
        zn = z / torch.sqrt(z.square().mean(-1, keepdim=True) + EPS) * w1
        r = x + sc * (g / (1 + torch.exp(-g))) * zn
        n = r / torch.sqrt(r.square().mean(-1, keepdim=True) + EPS) * w2

        def whole(v):
            return torch.zeros(B, T, D, dtype=v.dtype, device=v.device).masked_scatter(
                rows[..., None], v.detach())

        out = {"residual": whole(r), "normed": whole(n)}
        if case["train"]:
            grads = torch.autograd.grad(
                (r, n), full, (s["grad_residual"].double()[rows], s["grad_normed"].double()[rows]))
            keys = ("grad_residual", "grad_branch", "grad_gate", "grad_branch_weight",
                    "grad_scale", "grad_next_weight")
            out.update(zip(keys, grads))
    return out


def _exact_stored(s):
    x = s["x"].double()
    B, T, D = x.shape
    if s["lengths"] is not None:
        t = torch.arange(T, device=x.device)
        x = x.masked_fill((t[None] >= s["lengths"][:, None]).unsqueeze(-1), 0.0)
    top = torch.finfo(s["x"].dtype).max
    out = torch.empty_like(x)
    for at in range(0, D, GROUP):
        v = x[..., at:at + GROUP]
        amax = v.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(amax / 127)).clamp(min=-126)
        e = torch.where(amax > 127 * torch.exp2(e), e + 1, e)
        e = torch.where((amax <= 127 * torch.exp2(e - 1)) & (e > -126), e - 1, e)
        unit = torch.exp2(e)
        most = torch.floor(top / unit)
        out[..., at:at + GROUP] = torch.round(v / unit).clamp(min=-most, max=most) * unit
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "step":
            g = s["gate"].double()
            h = s["state"].double() / (1 + torch.exp(-g)) + s["x"].double() / (1 + torch.exp(g))
            return {"h": h, "state": h.clone()}
        if op == "scan":
            return _exact_scan(s)
        if op == "norm":
            return _exact_norm(s)
        stored = _exact_stored(s)
        if op == "pack":
            return {"x": stored}
        dy = s["grad_output"].double()
        if s["lengths"] is not None:
            t = torch.arange(dy.shape[1], device=dy.device)
            dy = dy.masked_fill((t[None] >= s["lengths"][:, None]).unsqueeze(-1), 0.0)
        return {"grad_weight": torch.einsum("btm,btd->md", dy, stored)}
