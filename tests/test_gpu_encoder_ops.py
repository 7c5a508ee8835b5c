"""The encoder operators against their formulas in float64.

Every bound is one rounding of the output's type plus the float32 error that
the operation count allows (see encoder_reference); inputs in masked places
are NaN or infinite throughout.
"""

import ctypes

import pytest
import torch

import encoder_reference as ref
from encoder_reference import TINY, U32, UNIT, assert_within

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


def _dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _gen(seed):
    return torch.Generator(device=_dev()).manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    v = torch.randn(*shape, generator=gen, device=_dev()) * scale + shift
    return v.to(dtype)


def _ragged(B, T):
    """Lengths that hold 0, 1 and T among them."""
    n = [(T * (k + 1)) // B for k in range(B)]
    n[0] = T
    if B > 1:
        n[-1] = 0
    if B > 2:
        n[-2] = min(1, T)
    return torch.tensor(n)


def _spoil(t, lengths, how):
    """Garbage past each length."""
    if lengths is None:
        return t
    live = ref.live_mask(lengths, t.shape[0], t.shape[1]).to(t.device)[..., None]
    return torch.where(live, t, torch.full_like(t, how))


# ---------------------------------------------------------------------------
# gated linear recurrence
# ---------------------------------------------------------------------------
def _recurrence_bounds(want, x, initial, dtype, T, grads=None):
    """Per output: u |value| + c T u32 A, A the largest magnitude that enters."""
    A = float(x.abs().max()) if x.numel() else 0.0
    if initial is not None:
        A = max(A, float(initial.detach().abs().max()))
    acc = 8 * T * U32 * A
    tol = {"h": UNIT[dtype] * want["h"].abs() + acc + TINY[dtype],
           "state": UNIT[torch.float32] * want["state"].abs() + acc}
    if "grad_x" in want:
        # lam sums at most the whole of dh; every link of either chain is off by 8 u32
        lam = float(grads)
        tol["grad_x"] = UNIT[dtype] * want["grad_x"].abs() + 8 * T * U32 * lam + TINY[dtype]
        tol["grad_gate"] = (UNIT[dtype] * want["grad_gate"].abs() + 24 * T * U32 * lam * A
                            + TINY[dtype])
        tol["grad_initial"] = 8 * T * U32 * lam + torch.zeros_like(want["grad_initial"])
    return tol


def _lam_max(x, gate, lengths, reverse, grad_h, grad_state):
    """A bound of |lam|: the recurrence of absolute gradients."""
    a = ref.recurrence(torch.zeros_like(x), gate, None, lengths, reverse,
                       None if grad_h is None else grad_h.abs(),
                       None if grad_state is None else grad_state.abs())
    i = torch.sigmoid(-ref.masked(gate, ref.live_mask(lengths, *x.shape[:2])))
    lam = torch.where(i > 0, a["grad_x"] / i.clamp_min(1e-300), torch.zeros_like(i))
    return max(float(lam.max()), float(a["grad_initial"].abs().max()))


def _check_recurrence(x, gate, initial, lengths, reverse, grad_h, grad_state):
    import torch_semimarkov_b200 as tsm

    T, dtype = x.shape[1], x.dtype
    leaves = [t.detach().requires_grad_(True) for t in (x, gate)]
    if initial is not None:
        initial = initial.detach().requires_grad_(True)
    h, state = tsm.gated_linear_recurrence(*leaves, initial, lengths, reverse=reverse)
    assert h.dtype == dtype and state.dtype == torch.float32
    want = ref.recurrence(x, gate, initial, lengths, reverse, grad_h, grad_state)
    outs, gouts = [], []
    if grad_h is not None:
        outs.append(h), gouts.append(grad_h)
    if grad_state is not None:
        outs.append(state), gouts.append(grad_state)
    inputs = leaves + ([initial] if initial is not None else [])
    grads = torch.autograd.grad(outs, inputs, gouts)
    live = ref.live_mask(lengths, *x.shape[:2])
    tol = _recurrence_bounds(want, ref.masked(x, live), initial, dtype, T,
                             _lam_max(x, gate, lengths, reverse, grad_h, grad_state))
    got = dict(h=h, state=state, grad_x=grads[0], grad_gate=grads[1])
    if initial is not None:
        got["grad_initial"] = grads[2]
    for k, v in got.items():
        assert_within(v, want[k], tol[k], k)
    # without gradients the same values come out
    with torch.no_grad():
        h2, s2 = tsm.gated_linear_recurrence(*leaves, initial, lengths, reverse=reverse)
    assert torch.equal(h, h2) and torch.equal(state, s2)
    return h, state, grads


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 63, 64, 65, 129, 300])
def test_recurrence_lengths_of_time(dtype, T):
    g = _gen(T)
    B, D = 3, 66
    x, gate = _normal(g, B, T, D, dtype=dtype), _normal(g, B, T, D, dtype=dtype, shift=2.0)
    s0 = _normal(g, B, D)
    _check_recurrence(x, gate, s0, None, T % 2 == 0, _normal(g, B, T, D, dtype=dtype),
                      _normal(g, B, D))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [1, 2, 3, 31, 64, 65, 130, 512])
@pytest.mark.parametrize("reverse", [False, True])
def test_recurrence_widths_and_ragged_lengths(dtype, D, reverse):
    g = _gen(D)
    B, T = 5, 75
    n = _ragged(B, T).to(_dev())
    x = _spoil(_normal(g, B, T, D, dtype=dtype), n, float("nan"))
    gate = _spoil(_normal(g, B, T, D, dtype=dtype, shift=1.0), n, float("inf"))
    dh = _spoil(_normal(g, B, T, D, dtype=dtype), n, float("-inf"))
    _check_recurrence(x, gate, _normal(g, B, D), n, reverse, dh, _normal(g, B, D))


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("T", [4097, 9000])
def test_recurrence_long(T, reverse):
    """Many chunks, memory that reaches across them (gates near one)."""
    g = _gen(T)
    B, D = 2, 34
    n = torch.tensor([T, T - 1500])
    x = _normal(g, B, T, D)
    gate = _normal(g, B, T, D, shift=7.0)
    _check_recurrence(x, gate, _normal(g, B, D), n, reverse, _normal(g, B, T, D),
                      _normal(g, B, D))


def test_recurrence_reads_slices_of_a_projection():
    """x and gate as slices of one (B, T, 3 D) tensor, a (T, B, D) order, and an
    odd offset that rules vectors out: strides, no copies."""
    g = _gen(4)
    B, T, D = 3, 70, 64
    wide = _normal(g, B, T, 3 * D + 1, dtype=torch.bfloat16)
    dh, ds = _normal(g, B, T, D, dtype=torch.bfloat16), _normal(g, B, D)
    _check_recurrence(wide[..., :D], wide[..., D:2 * D], None, None, False, dh, ds)
    _check_recurrence(wide[..., 1:D + 1], wide[..., 2 * D + 1:], None, None, True, dh, ds)
    swapped = _normal(g, T, B, 2 * D).transpose(0, 1)
    _check_recurrence(swapped[..., :D], swapped[..., D:], _normal(g, B, D), None, False,
                      dh.float().transpose(0, 1).contiguous().transpose(0, 1), None)
    columns = _normal(g, B, D, T).transpose(1, 2)  # channels not contiguous: copied
    _check_recurrence(columns, columns.flip(2), None, None, False, dh.float(), ds)


@pytest.mark.parametrize("which", ["h", "state"])
def test_recurrence_one_gradient_only(which):
    g = _gen(6)
    B, T, D = 2, 90, 20
    x, gate = _normal(g, B, T, D), _normal(g, B, T, D)
    _check_recurrence(x, gate, _normal(g, B, D), torch.tensor([90, 33]), False,
                      _normal(g, B, T, D) if which == "h" else None,
                      _normal(g, B, D) if which == "state" else None)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_recurrence_gates_at_their_limits(dtype):
    """Gates of plus and minus infinity, the type's largest and lowest value,
    and far into saturation: the state is kept or replaced exactly."""
    big = torch.finfo(dtype).max
    g = _gen(8)
    vals = torch.tensor([float("inf"), float("-inf"), big, -big, 90.0, -90.0, 0.0, 20.0])
    B, T, D = 1, 130, 8
    gate = vals[torch.randint(0, 8, (B, T, D), generator=torch.Generator().manual_seed(1))]
    gate = gate.to(_dev(), dtype)
    x = _normal(g, B, T, D, dtype=dtype)
    _check_recurrence(x, gate, _normal(g, B, D), None, False, _normal(g, B, T, D, dtype=dtype),
                      _normal(g, B, D))


def test_recurrence_all_masked_and_empty():
    import torch_semimarkov_b200 as tsm

    dev = _dev()
    nan = torch.full((2, 70, 6), float("nan"), device=dev)
    s0 = _normal(_gen(1), 2, 6)
    h, s = tsm.gated_linear_recurrence(nan, nan, s0, torch.tensor([0, 0]))
    assert torch.equal(h, torch.zeros_like(h)) and torch.equal(s, s0)
    i = s0.clone().requires_grad_(True)
    h, s = tsm.gated_linear_recurrence(nan, nan, i, torch.tensor([0, 0]))
    (gi,) = torch.autograd.grad(s, i, 2 * s0)
    assert torch.equal(gi, 2 * s0)
    x = torch.empty(2, 0, 6, device=dev, requires_grad=True)
    i = s0.clone().requires_grad_(True)
    h, s = tsm.gated_linear_recurrence(x, x, i)
    assert h.shape == (2, 0, 6) and torch.equal(s, s0)
    (gi,) = torch.autograd.grad(s, i, s0)
    assert torch.equal(gi, s0)
    h, s = tsm.gated_linear_recurrence(torch.empty(0, 5, 6, device=dev),
                                       torch.empty(0, 5, 6, device=dev))
    assert h.shape == (0, 5, 6) and s.shape == (0, 6)


def test_recurrence_gradient_against_differences():
    """The directional derivative against central differences of the kernel's
    own float32 forward.  Bound: rounding of the two losses over 2 eps (each
    output off by 8 T u32 A), plus twice the truncation that the float64 form
    shows for the same eps."""
    import torch_semimarkov_b200 as tsm

    g = _gen(12)
    B, T, D, eps = 2, 40, 6, 1e-2
    n = torch.tensor([40, 17])
    base = [_normal(g, B, T, D), _normal(g, B, T, D), _normal(g, B, D)]
    step = [_normal(g, *t.shape) for t in base]
    wh, ws = _normal(g, B, T, D), _normal(g, B, D)

    def loss(ts):
        h, s = tsm.gated_linear_recurrence(*ts, n)
        return float((h.double() * wh).sum() + (s.double() * ws).sum())

    def loss64(ts):
        o = ref.recurrence(*ts, n, False)
        return float((o["h"] * wh.cpu()).sum() + (o["state"] * ws.cpu()).sum())

    leaves = [t.clone().requires_grad_(True) for t in base]
    grads = torch.autograd.grad(tsm.gated_linear_recurrence(*leaves, n), leaves, (wh, ws))
    slope = sum(float((a.double() * b).sum()) for a, b in zip(grads, step))
    plus = [t + eps * d for t, d in zip(base, step)]
    minus = [t - eps * d for t, d in zip(base, step)]
    diff = (loss(plus) - loss(minus)) / (2 * eps)
    want = ref.recurrence(*base, n, False, wh, ws)
    slope64 = sum(float((want[k] * d.cpu()).sum())
                  for k, d in zip(("grad_x", "grad_gate", "grad_initial"), step))
    cut = abs((loss64(plus) - loss64(minus)) / (2 * eps) - slope64)
    A = max(float(t.abs().max()) for t in (base[0], base[2]))
    rounding = 8 * T * U32 * A * float(wh.abs().sum() + ws.abs().sum()) / eps
    assert abs(slope - diff) <= rounding + 2 * cut + 1e-3 * abs(slope64)
    assert abs(slope - slope64) <= 24 * T * U32 * A * float(wh.abs().sum()) * 4


def test_recurrence_is_reproducible_and_stream_ordered():
    import torch_semimarkov_b200 as tsm

    g = _gen(20)
    B, T, D = 2, 5000, 96
    x = _normal(g, B, T, D, dtype=torch.bfloat16).requires_grad_(True)
    gate = _normal(g, B, T, D, dtype=torch.bfloat16, shift=3.0).requires_grad_(True)
    dh = _normal(g, B, T, D, dtype=torch.bfloat16)

    def once():
        h, s = tsm.gated_linear_recurrence(x, gate)
        return (h, s, *torch.autograd.grad(h, (x, gate), dh))

    first = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    for _ in range(5):
        for a, b in zip(first, once()):
            assert torch.equal(a, b)


def test_recurrence_offsets_past_32_bits():
    """Rows that lie more than 2^31 elements apart."""
    import torch_semimarkov_b200 as tsm

    T, D, far = 3, 8, (1 << 30) + 8
    store = torch.empty(2 * far + D, dtype=torch.bfloat16, device=_dev())
    x = store.as_strided((1, T, D), (0, far, 1))
    small = _normal(_gen(3), 1, T, D, dtype=torch.bfloat16)
    x.copy_(small)
    gate = _normal(_gen(4), 1, T, D, dtype=torch.bfloat16)
    a = tsm.gated_linear_recurrence(x, gate)
    b = tsm.gated_linear_recurrence(small, gate)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    a = tsm.pack_activation(x)
    b = tsm.pack_activation(small)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("B,D", [(1, 1), (1, 64), (5, 66), (7, 63), (300, 512)])
def test_recurrence_step(dtype, B, D):
    import torch_semimarkov_b200 as tsm

    g = _gen(B + D)
    wide = _normal(g, B, 2 * D, dtype=dtype)
    x, gate, s = wide[:, :D], wide[:, D:], _normal(g, B, D)
    want = ref.recurrence(x[:, None], gate[:, None], s, None, False)
    tol = _recurrence_bounds(want, x, s, dtype, 1)
    h, out = tsm.gated_linear_recurrence_step(x, gate, s)
    assert_within(h[:, None], want["h"], tol["h"], "h")
    assert_within(out, want["state"], tol["state"], "state")
    # the full form over one position gives the same
    h1, s1 = tsm.gated_linear_recurrence(x[:, None], gate[:, None], s)
    assert torch.equal(h, h1[:, 0]) and torch.equal(out, s1)
    # in place, some streams idle with garbage in their inputs
    active = torch.arange(B, device=_dev()) % 3 != 1
    xs = torch.where(active[:, None], x, torch.full_like(x, float("nan")))
    mine = s.clone()
    h2, out2 = tsm.gated_linear_recurrence_step(xs, gate, mine, active, out_state=mine)
    assert out2 is mine
    assert torch.equal(mine, torch.where(active[:, None], out, s))
    assert torch.equal(h2, torch.where(active[:, None], h, torch.zeros_like(h)))


def test_step_in_a_cuda_graph():
    import torch_semimarkov_b200 as tsm

    g = _gen(2)
    B, D, n = 4, 64, 5
    xs, gs = _normal(g, n, B, D), _normal(g, n, B, D)
    x, gate, state = xs[0].clone(), gs[0].clone(), torch.zeros(B, D, device=_dev())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tsm.gated_linear_recurrence_step(x, gate, state.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, _ = tsm.gated_linear_recurrence_step(x, gate, state, out_state=state)
    want, s = tsm.gated_linear_recurrence(xs.transpose(0, 1), gs.transpose(0, 1))
    for t in range(n):
        x.copy_(xs[t]), gate.copy_(gs[t])
        graph.replay()
        tol = torch.full((B, D), 8 * n * U32 * float(xs.abs().max()), dtype=torch.float64)
        assert_within(h, want[:, t].cpu().double(), tol, f"h[{t}]")
    assert_within(state, s.cpu().double(), tol, "state")


# ---------------------------------------------------------------------------
# gated residual norm
# ---------------------------------------------------------------------------
def _norm_inputs(g, B, T, D, dtype, lengths=None):
    t = {"residual": _normal(g, B, T, D, dtype=dtype, scale=2.0),
         "branch": _normal(g, B, T, D, dtype=dtype, scale=0.5),
         "gate": _normal(g, B, T, D, dtype=dtype)}
    for k, how in zip(t, (float("nan"), float("inf"), float("-inf"))):
        t[k] = _spoil(t[k], lengths, how)
    w = {"w1": _normal(g, D, scale=0.2, shift=1.0), "scale": _normal(g, D, scale=0.2, shift=0.3),
         "w2": _normal(g, D, scale=0.2, shift=1.0)}
    return t, w


def _check_norm(t, w, lengths, grad_r, grad_n, eps=1e-6):
    """Bounds.  A row's sum of D terms is off by at most (16 + 10) u32 of the sum
    of magnitudes (16 in a lane, then a tree over lanes and warps), so both
    statistics by under 32 u32 and each output by 64 u32 of what enters it; a
    gradient passes two such rows and the recomputed r: 256.  Weight gradients
    add N rows one after another in the worst order."""
    import torch_semimarkov_b200 as tsm

    dtype = t["residual"].dtype
    B, T, D = t["residual"].shape
    leaves = [v.detach().requires_grad_(True) for v in (*t.values(), *w.values())]
    r, n = tsm.gated_residual_norm(*leaves, lengths=lengths, eps=eps)
    want = ref.block_norm(*t.values(), *w.values(), lengths, eps, grad_r, grad_n)
    u = UNIT[dtype]
    rows = want["r"].abs().amax(-1, keepdim=True) + ref.masked(
        t["residual"], ref.live_mask(lengths, B, T)).abs().amax(-1, keepdim=True)
    assert_within(r, want["r"], u * want["r"].abs() + 64 * U32 * rows + TINY[dtype], "r")
    rr = torch.where(rows > 0, want["n"].abs().amax(-1, keepdim=True), rows)
    assert_within(n, want["n"], u * want["n"].abs() + 128 * U32 * (rr + 1) * 8 + TINY[dtype], "n")
    outs = [(o, g) for o, g in ((r, grad_r), (n, grad_n)) if g is not None]
    got = torch.autograd.grad([o for o, _ in outs], leaves, [g for _, g in outs])
    for v, k in zip(got[:3], ("dx", "dz", "dg")):
        mag = want["abs_" + k].amax(-1, keepdim=True)
        assert v.dtype == dtype
        assert_within(v, want[k], u * want[k].abs() + 256 * U32 * mag + TINY[dtype], k)
    N = B * T
    for v, k in zip(got[3:], ("dw1", "ds", "dw2")):
        assert v.dtype == torch.float32
        assert_within(v, want[k], (N + 256) * U32 * want["abs_" + k] + 1e-30, k)
    with torch.no_grad():
        r2, n2 = tsm.gated_residual_norm(*leaves, lengths=lengths, eps=eps)
    assert torch.equal(r, r2) and torch.equal(n, n2)
    return r, n, got


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [1, 3, 8, 31, 64, 203, 256, 257, 512, 520, 1000, 1024, 1025, 2048,
                               4096, 4100, 8192])
def test_norm_widths(dtype, D):
    g = _gen(D)
    B, T = 3, 7
    n = _ragged(B, T).to(_dev()) if D % 2 else None
    t, w = _norm_inputs(g, B, T, D, dtype, n)
    dr = _spoil(_normal(g, B, T, D, dtype=dtype), n, float("nan"))
    dn = _spoil(_normal(g, B, T, D, dtype=dtype), n, float("inf"))
    _check_norm(t, w, n, dr, dn)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [4, 8, 16, 24, 32, 40, 56, 64, 72, 120, 128, 136, 640, 768, 776, 1280,
                               1536])
def test_norm_rows_that_share_a_warp(dtype, D):
    """Rows of every length of the lanes that a row takes; sequences that end
    in the middle of a warp's rows; the checkpoint written beside them."""
    import torch_semimarkov_b200 as tsm

    g = _gen(D + 7)
    B, T = 5, 37
    n = torch.tensor([37, 0, 18, 1, 36], device=_dev())
    t, w = _norm_inputs(g, B, T, D, dtype, n)
    dr = _spoil(_normal(g, B, T, D, dtype=dtype), n, float("nan"))
    dn = _spoil(_normal(g, B, T, D, dtype=dtype), n, float("inf"))
    _check_norm(t, w, n, dr, dn)
    _, y, p = tsm.gated_residual_norm(*t.values(), *w.values(), lengths=n, pack=True)
    q = tsm.pack_activation(y)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
    y, p = tsm.rms_norm(t["residual"], w["w2"], n, pack=True)
    q = tsm.pack_activation(y)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [2, 29, 37, 61, 65, 100])
def test_norm_narrow_rows_without_alignment(dtype, D):
    import torch_semimarkov_b200 as tsm

    g = _gen(D + 11)
    B, T = 5, 37
    n = torch.tensor([37, 0, 18, 1, 36], device=_dev())
    t, w = _norm_inputs(g, B, T, D, dtype, n)
    dr = _spoil(_normal(g, B, T, D, dtype=dtype), n, float("nan"))
    dn = _spoil(_normal(g, B, T, D, dtype=dtype), n, float("inf"))
    _check_norm(t, w, n, dr, dn)
    _, y, p = tsm.gated_residual_norm(*t.values(), *w.values(), lengths=n, pack=True)
    q = tsm.pack_activation(y)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("B,T", [(1, 1), (1, 5), (2, 1500), (40, 60)])
def test_norm_row_counts(dtype, B, T):
    g = _gen(B * T)
    D = 40
    t, w = _norm_inputs(g, B, T, D, dtype)
    _check_norm(t, w, None, _normal(g, B, T, D, dtype=dtype), _normal(g, B, T, D, dtype=dtype))


@pytest.mark.parametrize("which", ["r", "n"])
def test_norm_one_gradient_only(which):
    g = _gen(3)
    B, T, D = 2, 9, 72
    t, w = _norm_inputs(g, B, T, D, torch.bfloat16)
    d = _normal(g, B, T, D, dtype=torch.bfloat16)
    _check_norm(t, w, None, d if which == "r" else None, d if which == "n" else None)


def test_norm_strides_and_reproducible():
    g = _gen(5)
    B, T, D = 3, 50, 64
    wide = _normal(g, B, T, 3 * D + 1, dtype=torch.bfloat16)
    w = _norm_inputs(g, 1, 1, D, torch.bfloat16)[1]
    dr, dn = _normal(g, B, T, D, dtype=torch.bfloat16), _normal(g, B, T, D, dtype=torch.bfloat16)
    for k in (0, 1):  # aligned slices, and slices at an odd offset
        t = {"residual": wide[..., k:D + k], "branch": wide[..., D + k:2 * D + k],
             "gate": wide[..., 2 * D + k:3 * D + k]}
        a = _check_norm(t, w, None, dr, dn)
        b = _check_norm({k2: v.contiguous() for k2, v in t.items()}, w, None, dr, dn)
        for u, v in zip((*a[:2], *a[2][:3]), (*b[:2], *b[2][:3])):
            # vector and single loads give a lane other channels: sums differ by rounding
            tol = 2 * UNIT[torch.bfloat16] * v.detach().cpu().double().abs() + 1e-4
            assert_within(u, v.detach().cpu().double(), tol, "strided")
        again = _check_norm(t, w, None, dr, dn)
        for u, v in zip((*a[:2], *a[2]), (*again[:2], *again[2])):
            assert torch.equal(u, v)


def test_norm_zero_rows_and_eps():
    """Rows of zeros: rms is sqrt(eps), gradients are finite."""
    g = _gen(7)
    B, T, D = 1, 4, 48
    t, w = _norm_inputs(g, B, T, D, torch.float32)
    for k in t:
        t[k][:, 1:3] = 0.0
    _check_norm(t, w, None, _normal(g, B, T, D), _normal(g, B, T, D), eps=1e-2)


def test_norm_gradients_by_differentiation():
    """The formula's gradients against automatic differentiation of the float64 forward."""
    g = torch.Generator().manual_seed(1)
    B, T, D, eps = 2, 3, 10, 1e-5
    full = [torch.randn(B, T, D, generator=g, dtype=torch.float64) for _ in range(3)]
    full += [torch.randn(D, generator=g, dtype=torch.float64) for _ in range(3)]
    dr, dn = (torch.randn(B, T, D, generator=g, dtype=torch.float64) for _ in range(2))
    want = ref.block_norm(*full, None, eps, dr, dn)
    x, z, gt, w1, s, w2 = (v.requires_grad_(True) for v in full)
    b = z / torch.sqrt(z.square().mean(-1, keepdim=True) + eps) * w1
    r = x + s * torch.nn.functional.silu(gt) * b
    n = r / torch.sqrt(r.square().mean(-1, keepdim=True) + eps) * w2
    got = torch.autograd.grad((r, n), full, (dr, dn))
    for v, k in zip(got, ("dx", "dz", "dg", "dw1", "ds", "dw2")):
        torch.testing.assert_close(v, want[k], rtol=1e-11, atol=1e-11)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [5, 64, 203, 512, 3000])
def test_rms_norm(dtype, D):
    import torch_semimarkov_b200 as tsm

    g = _gen(D)
    B, T, eps = 3, 20, 1e-6
    n = _ragged(B, T)
    x = _spoil(_normal(g, B, T, D, dtype=dtype), n, float("nan")).requires_grad_(True)
    w = _normal(g, D, scale=0.3, shift=1.0).requires_grad_(True)
    dn = _normal(g, B, T, D, dtype=dtype)
    y = tsm.rms_norm(x, w, n, eps)
    want = ref.block_norm(x, None, None, None, None, w, n, eps, None, dn)
    gx, gw = torch.autograd.grad(y, (x, w), dn)
    u = UNIT[dtype]
    assert_within(y, want["n"], u * want["n"].abs() + 1024 * U32 * (1 + want["n"].abs().max()), "n")
    mag = want["abs_dx"].amax(-1, keepdim=True)
    assert_within(gx, want["dx"], u * want["dx"].abs() + 256 * U32 * mag + TINY[dtype], "dx")
    assert_within(gw, want["dw2"], (B * T + 256) * U32 * want["abs_dw2"] + 1e-30, "dw2")


def test_norm_empty():
    import torch_semimarkov_b200 as tsm

    dev = _dev()
    D = 8
    w = [torch.ones(D, device=dev, requires_grad=True) for _ in range(3)]
    for shape in ((0, 4, D), (3, 0, D)):
        t = [torch.empty(shape, device=dev, requires_grad=True) for _ in range(3)]
        r, n = tsm.gated_residual_norm(*t, *w)
        assert r.shape == n.shape == shape
        for v in torch.autograd.grad((r.sum() + n.sum()), w):
            assert torch.equal(v, torch.zeros(D, device=dev))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [1, 33, 64, 203, 512, 1100])
def test_norm_writes_the_checkpoint(dtype, D):
    """pack=True equals pack_activation of the rounded output, bit for bit."""
    import torch_semimarkov_b200 as tsm

    g = _gen(D)
    B, T = 3, 11
    n = _ragged(B, T)
    t, w = _norm_inputs(g, B, T, D, dtype, n)
    r, y, p = tsm.gated_residual_norm(*t.values(), *w.values(), lengths=n, pack=True)
    q = tsm.pack_activation(y)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
    y, p = tsm.rms_norm(t["residual"], w["w2"], n, pack=True)
    q = tsm.pack_activation(y)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)


# ---------------------------------------------------------------------------
# 8-bit checkpoints
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [1, 31, 32, 33, 64, 203, 512])
def test_pack_is_exact(dtype, D):
    import torch_semimarkov_b200 as tsm

    g = _gen(D)
    B, T = 4, 9
    n = _ragged(B, T)
    x = _normal(g, B, T, D, dtype=dtype) * torch.exp(_normal(g, B, T, 1, scale=3.0)).to(dtype)
    x = _spoil(x, n, float("nan"))
    p = tsm.pack_activation(x, n)
    codes, scales, values = ref.stored(x, n)
    assert torch.equal(p.codes.cpu(), codes) and torch.equal(p.scales.cpu(), scales)
    assert p.shape == x.shape
    assert torch.equal(p.unpack().cpu(), values.to(dtype))
    assert torch.equal(p.unpack(torch.float32).cpu().double(), values)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_pack_edges(dtype):
    """Ties, the step between scales, subnormal and largest values, zeros,
    infinities and NaN."""
    import torch_semimarkov_b200 as tsm

    top = torch.finfo(dtype).max
    tiny = TINY[dtype]
    rows = torch.zeros(12, 64)
    rows[0, :32] = torch.arange(32) - 16.5
    rows[0, 0] = 127.0
    rows[1, 0], rows[1, 5] = 127.5, -0.5
    rows[2, 3], rows[2, 4] = top, -top
    rows[3, 3] = -top
    rows[4, 1], rows[4, 2] = tiny, -3 * tiny
    rows[5, 40] = float("inf")
    rows[6, 2] = float("nan")
    rows[6, 40] = 2.0
    rows[7, 31], rows[7, 32] = 1.0, -1.0
    rows[8, :] = torch.linspace(-1, 1, 64)
    rows[9, 0], rows[9, 1] = 127 * 2.0 ** -3, 63.5 * 2.0 ** -3
    rows[10, 0] = float("-inf")
    x = rows.view(1, 12, 64).to(_dev(), dtype)
    p = tsm.pack_activation(x)
    codes, scales, values = ref.stored(x, None)
    assert torch.equal(p.codes.cpu(), codes) and torch.equal(p.scales.cpu(), scales)
    got = p.unpack().cpu()
    torch.testing.assert_close(got, values.to(dtype), rtol=0, atol=0, equal_nan=True)
    assert torch.isfinite(got[0, 2:5]).all()


def test_pack_strides_and_empty():
    import torch_semimarkov_b200 as tsm

    g = _gen(2)
    wide = _normal(g, 3, 20, 130, dtype=torch.bfloat16)
    for v in (wide[..., 2:66], wide[..., 1:65], wide.transpose(0, 1), wide[:, ::2, :96]):
        a, b = tsm.pack_activation(v), tsm.pack_activation(v.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    p = tsm.pack_activation(torch.empty(2, 0, 40, device=_dev()))
    assert p.unpack().shape == (2, 0, 40)


def _check_weight_grad(x, dy, lengths, dtype=None):
    """Products are exact (7-bit codes times a power of two, split dy), so the
    error is that of float32 sums: at most N u32 of the sum of magnitudes."""
    import torch_semimarkov_b200 as tsm

    p = tsm.pack_activation(x, lengths)
    got = tsm.packed_weight_grad(dy, p, lengths, dtype)
    dtype = dy.dtype if dtype is None else dtype
    assert got.dtype == dtype
    live = ref.live_mask(lengths, *x.shape[:2])
    v = ref.stored(x, lengths)[2].reshape(-1, x.shape[2])
    d = ref.masked(dy, live).reshape(-1, dy.shape[2])
    want, mag = d.t() @ v, d.abs().t() @ v.abs()
    N = max(1, v.shape[0])
    assert_within(got, want, UNIT[dtype] * want.abs() + N * U32 * mag + TINY[dtype], "dw")
    return got


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("B,T,D,M", [(1, 1, 1, 1), (1, 1, 32, 8), (2, 7, 40, 24), (3, 50, 203, 97),
                                     (4, 130, 64, 128), (1, 300, 256, 384), (2, 65, 130, 257),
                                     (5, 64, 33, 1), (1, 2000, 96, 64), (70, 3, 64, 136)])
def test_weight_grad(dtype, B, T, D, M):
    g = _gen(T + D + M)
    x, dy = _normal(g, B, T, D, dtype=dtype), _normal(g, B, T, M, dtype=dtype)
    a = _check_weight_grad(x, dy, None)
    b = _check_weight_grad(x, dy, None)
    assert torch.equal(a, b)
    n = _ragged(B, T)
    _check_weight_grad(_spoil(x, n, float("nan")), _spoil(dy, n, float("inf")), n, torch.float32)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_weight_grad_of_many_positions(dtype):
    g = _gen(1)
    B, T, D, M = 3, 5000, 128, 200
    n = torch.tensor([5000, 4099, 1])
    _check_weight_grad(_normal(g, B, T, D, dtype=dtype), _normal(g, B, T, M, dtype=dtype), None)
    _check_weight_grad(_normal(g, B, T, D, dtype=dtype), _normal(g, B, T, M, dtype=dtype), n)


@pytest.mark.parametrize("D,M", [(64, 72), (160, 264)])
def test_weight_grad_of_float16_from_end_to_end(D, M):
    """Groups of the smallest subnormal numbers, of the largest and of zeros,
    and gradients that are subnormal themselves."""
    g = _gen(D)
    B, T = 2, 333
    x, dy = (_normal(g, B, T, n, dtype=torch.float16) for n in (D, M))
    x[:, ::5] = x[:, ::5] * 2.0 ** -22
    x[:, 1::5, :32] = 65504.0
    x[:, 2::5, 32:] = 0.0
    x[:, 3::5] = x[:, 3::5] * 2.0 ** -12
    dy[:, ::3] = dy[:, ::3] * 2.0 ** -20
    n = torch.tensor([333, 100])
    _check_weight_grad(x, dy, None, torch.float32)
    _check_weight_grad(x, dy, n, torch.float32)


def test_weight_grad_of_float16_over_a_wider_checkpoint():
    """A checkpoint of bfloat16 values holds what float16 does not."""
    g = _gen(3)
    x = _normal(g, 2, 100, 64, dtype=torch.bfloat16) * 1e20
    x[:, ::2] *= 1e-30
    _check_weight_grad(x, _normal(g, 2, 100, 64, dtype=torch.float16), None, torch.float32)


def test_weight_grad_strides_and_scales():
    """grad_output as a slice (aligned and not) and transposed; scales far apart."""
    g = _gen(9)
    B, T, D, M = 2, 90, 64, 64
    x = _normal(g, B, T, D, dtype=torch.bfloat16) * torch.exp2(
        torch.randint(-20, 20, (B, T, 1), generator=g, device=_dev()).float()).to(torch.bfloat16)
    wide = _normal(g, B, T, 3 * M + 1, dtype=torch.bfloat16)
    for dy in (wide[..., M:2 * M], wide[..., 1:M + 1],
               _normal(g, T, B, M, dtype=torch.bfloat16).transpose(0, 1)):
        _check_weight_grad(x, dy, None, torch.float32)
    _check_weight_grad(x, wide[..., :M].float(), None)


def test_weight_grad_nonfinite_and_empty():
    """An input group that was not finite makes its channels' gradients NaN and
    no others; an infinite gradient stays where it belongs; no positions, no gradient."""
    import torch_semimarkov_b200 as tsm

    g = _gen(14)
    B, T, D, M = 1, 70, 96, 40
    x, dy = _normal(g, B, T, D), _normal(g, B, T, M)
    x[0, 5, 40] = float("inf")
    w = tsm.packed_weight_grad(dy, tsm.pack_activation(x))
    assert torch.isnan(w[:, 32:64]).all()
    assert torch.isfinite(w[:, :32]).all() and torch.isfinite(w[:, 64:]).all()
    x[0, 5, 40] = 0.0
    dy[0, 66, 3] = float("inf")
    w = tsm.packed_weight_grad(dy, tsm.pack_activation(x))
    assert not torch.isfinite(w[3]).any()
    rest = torch.cat([w[:3], w[4:]])
    assert torch.isfinite(rest).all()
    empty = tsm.packed_weight_grad(dy[:, :0], tsm.pack_activation(x[:, :0]))
    assert torch.equal(empty, torch.zeros(M, D, device=_dev()))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_packed_linear(dtype):
    import torch_semimarkov_b200 as tsm

    g = _gen(30)
    B, T, D, M = 3, 40, 64, 48
    n = torch.tensor([40, 11, 0])
    x = _spoil(_normal(g, B, T, D, dtype=dtype), n, 0.0).requires_grad_(True)
    w = _normal(g, M, D, scale=0.1).requires_grad_(True)
    b = _normal(g, M).requires_grad_(True)
    dy = _normal(g, B, T, M, dtype=dtype)
    y = tsm.packed_linear(x, w, b, lengths=n)
    plain = (x @ w.to(dtype).t()) + b.to(dtype)
    torch.testing.assert_close(y, plain, rtol=2 * UNIT[dtype] + 1e-5, atol=4 * UNIT[dtype])
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy)
    assert gw.dtype == torch.float32 and gx.dtype == dtype
    torch.testing.assert_close(gx, dy @ w.to(dtype), rtol=2 * UNIT[dtype] + 1e-5,
                               atol=4 * UNIT[dtype])
    p = tsm.pack_activation(x, n)
    assert torch.equal(gw, tsm.packed_weight_grad(dy, p, n, torch.float32))
    live = ref.live_mask(n, B, T).to(_dev())[..., None]
    torch.testing.assert_close(gb, (dy.float() * live).sum((0, 1)), rtol=1e-5, atol=1e-4)
    y2 = tsm.packed_linear(x, w, packed=p, lengths=n)
    (gw2,) = torch.autograd.grad(y2, w, dy)
    assert torch.equal(gw, gw2)


def test_calls_from_a_thread_without_a_context():
    """As in autograd's worker threads: nothing in a call before the kernel's
    launch may rely on a CUDA context that is current already."""
    import threading

    import torch_semimarkov_b200 as tsm

    g = _gen(40)
    x = _normal(g, 4, 10, 512, dtype=torch.bfloat16)
    leaf = x.clone().requires_grad_(True)

    def call():
        h, _ = tsm.gated_linear_recurrence(leaf, leaf)
        gx, = torch.autograd.grad(h, leaf, x)
        w = tsm.packed_weight_grad(x, tsm.pack_activation(x))
        return h.detach(), gx, w

    for _ in range(3):
        want = call()  # fills the allocator, so that the thread allocates nothing
        got = []
        t = threading.Thread(target=lambda: got.append(call()))
        t.start()
        t.join()
        for a, b in zip(want, got[0]):
            assert torch.equal(a, b)
        del got


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals_on_the_gpu():
    import torch_semimarkov_b200 as tsm

    dev = _dev()
    x = torch.zeros(2, 5, 8, device=dev)
    with pytest.raises(ValueError, match="gate"):
        tsm.gated_linear_recurrence(x, x[:, :4])
    with pytest.raises(ValueError, match="gate"):
        tsm.gated_linear_recurrence(x, x.half())
    with pytest.raises(RuntimeError, match="CUDA"):
        tsm.gated_linear_recurrence(x, x.cpu())
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        tsm.gated_linear_recurrence(x.double(), x.double())
    with pytest.raises(ValueError, match="initial_state"):
        tsm.gated_linear_recurrence(x, x, torch.zeros(8, device=dev))
    with pytest.raises(ValueError, match="lengths"):
        tsm.gated_linear_recurrence(x, x, lengths=torch.tensor([5]))
    with pytest.raises(ValueError, match="lengths"):
        tsm.gated_linear_recurrence(x, x, lengths=torch.tensor([5, 6]))
    with pytest.raises(ValueError, match="state"):
        tsm.gated_linear_recurrence_step(x[:, 0], x[:, 0], x[:, 0].half())
    with pytest.raises(ValueError, match="active"):
        tsm.gated_linear_recurrence_step(x[:, 0], x[:, 0], x[:, 0].contiguous(),
                                         torch.zeros(3, dtype=torch.bool, device=dev))
    w = torch.ones(8, device=dev)
    with pytest.raises(ValueError, match="branch"):
        tsm.gated_residual_norm(x, None, None, w, w, w)
    with pytest.raises(ValueError, match="residual_scale"):
        tsm.gated_residual_norm(x, x, x, w, w[:4], w)
    with pytest.raises(ValueError, match="eps"):
        tsm.rms_norm(x, w, eps=-1.0)
    with pytest.raises(NotImplementedError):
        big = torch.zeros(1, 1, 8200, device=dev)
        tsm.rms_norm(big, torch.ones(8200, device=dev))
    p = tsm.pack_activation(x)
    with pytest.raises(ValueError, match="packed"):
        tsm.packed_weight_grad(torch.zeros(2, 4, 3, device=dev), p)
    with pytest.raises(ValueError, match="layout"):
        tsm.PackedActivation(p.codes[:, :, :16], p.scales, 8, torch.float32).unpack()
    with pytest.raises(ValueError, match="weight"):
        tsm.packed_linear(x, torch.zeros(3, 7, device=dev))
    with pytest.raises(ValueError, match="packed"):
        tsm.packed_linear(x, torch.zeros(3, 8, device=dev, requires_grad=True),
                          packed=tsm.pack_activation(x[:, :3]))


def test_workspace_too_small_is_refused():
    """Through the C ABI: a short workspace is an error code, nothing is launched."""
    from torch_semimarkov_b200 import _lib

    lib = _lib.load()
    x = torch.zeros(2, 5, 8, device=_dev())
    p = _lib._recurrence(x, x, None, None, False)
    s = torch.zeros(2, 8, device=_dev())
    need = lib.semicrf_recurrence_workspace_size(p)
    ws = torch.empty(need, dtype=torch.uint8, device=_dev())
    st = lib.semicrf_recurrence_forward(p, _lib._sequence(x), s.data_ptr(), None, ws.data_ptr(),
                                        need - 1, ctypes.c_void_p(0))
    assert st == _lib.SEMICRF_ERR_WORKSPACE
