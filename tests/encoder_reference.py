"""Plain float64 forms of the encoder operators, written from their formulas,
and the error bounds that the tests hold the kernels to.

Rounding: an output of type t is rounded once, by at most u(t) |value|.  What
the kernels compute before that is float32: a chain of n dependent operations
on magnitudes of at most A is off by at most about c n u32 A, with c the
operations of a link (sigmoid, two products and a sum: 8 covers them).
"""

import torch

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# spacing of the subnormal numbers: the rounding error next to zero
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
GROUP = 32


def live_mask(lengths, B, T):
    if lengths is None:
        return torch.ones(B, T, dtype=torch.bool)
    return torch.arange(T)[None] < lengths.cpu()[:, None]


def masked(v, live):
    """v in float64 on the CPU, zeros in place of the positions that are not live."""
    v = v.detach().cpu().double()
    return torch.where(live[..., None], v, torch.zeros_like(v))


def recurrence(x, gate, initial, lengths, reverse, grad_h=None, grad_state=None):
    """Position by position: dict of h, state and (with grad_h) the gradients."""
    B, T, D = x.shape
    live = live_mask(lengths, B, T)
    x, g = masked(x, live), masked(gate, live)
    f, i = torch.sigmoid(g), torch.sigmoid(-g)
    s = torch.zeros(B, D, dtype=torch.float64) if initial is None else initial.detach().cpu().double()
    order = range(T - 1, -1, -1) if reverse else range(T)
    h = torch.zeros(B, T, D, dtype=torch.float64)
    before = torch.zeros_like(h)
    for t in order:
        before[:, t] = s
        new = f[:, t] * s + i[:, t] * x[:, t]
        s = torch.where(live[:, t, None], new, s)
        h[:, t] = torch.where(live[:, t, None], s, torch.zeros_like(s))
    out = {"h": h, "state": s}
    if grad_h is None and grad_state is None:
        return out
    dh = torch.zeros_like(h) if grad_h is None else masked(grad_h, live)
    lam = torch.zeros(B, D, dtype=torch.float64) if grad_state is None else \
        grad_state.detach().cpu().double()
    dx, dg = torch.zeros_like(h), torch.zeros_like(h)
    for t in reversed(order):
        on = live[:, t, None]
        at = lam + dh[:, t]
        dx[:, t] = torch.where(on, at * i[:, t], torch.zeros_like(at))
        dg[:, t] = torch.where(on, at * (before[:, t] - x[:, t]) * f[:, t] * i[:, t],
                               torch.zeros_like(at))
        lam = torch.where(on, at * f[:, t], lam)
    out.update(grad_x=dx, grad_gate=dg, grad_initial=lam)
    return out


def block_norm(residual, branch, gate, w1, scale, w2, lengths, eps, grad_r=None, grad_n=None):
    """Forward by the formula; gradients by the formula too (see gradients_by_autograd)."""
    B, T, D = residual.shape
    live = live_mask(lengths, B, T)
    x = masked(residual, live)
    w1, scale, w2 = (None if w is None else w.detach().cpu().double() for w in (w1, scale, w2))
    if branch is not None:
        z, g = masked(branch, live), masked(gate, live)
        rz = 1 / torch.sqrt(z.square().mean(-1, keepdim=True) + eps)
        zh = z * rz
        sig = torch.sigmoid(g)
        u = g * sig
        r = x + scale * u * zh * w1
    else:
        r = x
    rr = 1 / torch.sqrt(r.square().mean(-1, keepdim=True) + eps)
    rh = r * rr
    zero = torch.zeros_like(r)
    n = torch.where(live[..., None], rh * w2, zero)
    out = {"r": torch.where(live[..., None], r, zero), "n": n}
    if grad_r is None and grad_n is None:
        return out
    dr = zero if grad_r is None else masked(grad_r, live)
    dn = zero if grad_n is None else masked(grad_n, live)
    p = dn * w2
    d = dr + rr * (p - rh * (p * rh).mean(-1, keepdim=True))
    mag = dr.abs() + rr * (p.abs() + rh.abs() * (p * rh).abs().mean(-1, keepdim=True))
    out.update(dx=d, dw2=(dn * rh).sum((0, 1)), abs_dx=mag, abs_dw2=(dn * rh).abs().sum((0, 1)))
    if branch is not None:
        db = d * scale * u
        q = db * w1
        adb = mag * (scale * u).abs()
        aq = adb * w1.abs()
        out.update(
            dz=rz * (q - zh * (q * zh).mean(-1, keepdim=True)),
            abs_dz=rz * (aq + zh.abs() * (aq * zh.abs()).mean(-1, keepdim=True)),
            dg=d * scale * zh * w1 * sig * (1 + g * (1 - sig)),
            abs_dg=mag * (scale * zh * w1).abs() * (sig * (1 + g.abs())),
            dw1=(db * zh).sum((0, 1)), abs_dw1=(adb * zh.abs()).sum((0, 1)),
            ds=(d * u * zh * w1).sum((0, 1)), abs_ds=(mag * (u * zh * w1).abs()).sum((0, 1)))
    return out


def stored(x, lengths):
    """(codes, scale bytes, values) of the 8-bit checkpoint of x, in float64 and
    by searching e upwards rather than from the bits of the maximum."""
    B, T, D = x.shape
    live = live_mask(lengths, B, T)
    v = masked(x, live)
    top = float(torch.finfo(x.dtype).max)
    G = -(-D // GROUP)
    v = torch.nn.functional.pad(v, (0, G * GROUP - D)).view(B, T, G, GROUP)
    amax = v.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(v).all(-1, keepdim=True)
    e = torch.full_like(amax, -126)
    for k in range(-126, 123):
        e = torch.where(amax > 127 * 2.0 ** k, torch.full_like(e, k + 1), e)
    unit = torch.exp2(e)
    most = torch.floor(top / unit)
    q = torch.round(v / unit)
    q = torch.minimum(torch.maximum(q, -most), most)
    q = torch.where(finite, q, torch.zeros_like(q))
    byte = torch.where(amax == 0, torch.zeros_like(e), e + 127)
    byte = torch.where(finite, byte, torch.full_like(e, 255))
    values = torch.where(finite, q * unit, torch.full_like(q, float("nan")))
    return (q.view(B, T, G * GROUP).to(torch.int8), byte[..., 0].to(torch.uint8),
            values.view(B, T, G * GROUP)[..., :D])


def assert_within(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities differ"
    err = (got - want).abs()
    bad = (err > tol) & ~nan & ~inf
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: "
                             f"got {got[i]!r}, want {want[i]!r}, bound {tol.expand_as(err)[i]:.3e}")
