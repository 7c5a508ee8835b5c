"""The encoder operators where their rules meet their limits: long sums,
tensors whose rows overlap, gates and states at the ends of their types.

Bounds follow from the operation count, as in encoder_reference."""

import pytest
import torch

import encoder_reference as ref

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


def _offset(t):
    """The same values in rows that do not start on 16-byte boundaries."""
    wide = torch.empty(*t.shape[:-1], t.shape[-1] + 1, dtype=t.dtype, device=t.device)
    wide[..., 1:] = t
    return wide[..., 1:]


# ---------------------------------------------------------------------------
# weight gradient: sums of many positions
# ---------------------------------------------------------------------------
# Forms: rows of 16-bit types on 16-byte boundaries (bulk copies), others,
# float16 over a checkpoint of another type (two pieces), float32 (three).
FORMS = [("bf16", torch.bfloat16, True), ("bf16 unaligned", torch.bfloat16, False),
         ("fp16", torch.float16, True), ("fp16 unaligned", torch.float16, False),
         ("fp32", torch.float32, True), ("fp32 unaligned", torch.float32, False)]


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("M,D", [(2000, 1000), (1000, 500), (120, 96)])
@pytest.mark.parametrize("form", FORMS, ids=[f[0] for f in FORMS])
def test_weight_grad_sums_every_position_once(form, M, D, ragged):
    """Values whose sums float32 holds exactly, in any order: not one position
    may be missing or counted twice.  Runs of several thousand positions pass
    through every slot and both halves of tensor memory several times.

    16 bits: integers, at most 15,000 * 3 * 4 < 2^24.  float32: multiples of
    2^-15 that need all three pieces (leading, 2^-7 and 2^-15), summed over
    every 32nd channel value, so that sums stay below 2^9."""
    import torch_semimarkov_b200 as tsm

    _, dtype, aligned = form
    g = _gen(M + ragged)
    B, T = 3, 5000
    sign = 1 - 2 * torch.randint(0, 2, (B, T, D), generator=g, device=_dev()).float()
    if dtype == torch.float32:
        some = torch.randint(0, 32, (B, T, D), generator=g, device=_dev()) == 0
        x = sign * some
        a, b, c = (torch.randint(lo, hi, (B, T, M), generator=g, device=_dev()).float()
                   for lo, hi in ((1, 4), (0, 2), (0, 2)))
        dy = a + b * 2.0 ** -7 + c * 2.0 ** -15
    else:
        x = sign * 2.0 ** torch.randint(0, 3, (B, T, D), generator=g, device=_dev())
        dy = torch.randint(-3, 4, (B, T, M), generator=g, device=_dev()).float()
    x, dy = x.to(dtype), dy.to(dtype)
    n = torch.tensor([T, 4111, 0], device=_dev()) if ragged else None
    p = tsm.pack_activation(x, n)
    assert n is not None or torch.equal(p.unpack(), x)
    got = tsm.packed_weight_grad(dy if aligned else _offset(dy), p, n, torch.float32)
    live = torch.ones(B, T, 1, device=_dev()) if n is None else \
        (torch.arange(T, device=_dev()) < n[:, None]).float()[..., None]
    want = torch.matmul((dy.double() * live).view(-1, M).t(), x.double().view(-1, D))
    if dtype == torch.float32:
        assert float(want.abs().max()) < 2.0 ** 8  # and every part of a sum below 2^9
    assert torch.equal(got.double(), want)


LONG = [("bf16", torch.bfloat16, torch.bfloat16, True),
        ("bf16 unaligned", torch.bfloat16, torch.bfloat16, False),
        ("fp16", torch.float16, torch.float16, True),
        ("fp16 over bf16", torch.float16, torch.bfloat16, True),
        ("fp32", torch.float32, torch.float32, True)]


@pytest.mark.parametrize("form", LONG, ids=[f[0] for f in LONG])
def test_weight_grad_of_one_sign_does_not_shrink(form):
    """131,072 positions of positive values in one run: the tensor cores' sums
    truncate, always downwards, so the error may only be that of a segment.

    Bound, of the result: a sum of 2,048 positions (512 for float32) grows
    evenly through 128 (32) truncations for each piece, each at most 2^-23 of
    what has been summed, half the final on average; the segments' sum rounds
    as often as there are segments, at most 2^-24 of half the final on average.
    A tenth is added for sums that do not grow quite evenly."""
    import torch_semimarkov_b200 as tsm

    _, dtype, stored, aligned = form
    g = _gen(7)
    N, D, M = 131072, 1024, 2560
    x = torch.rand(1, N, D, generator=g, device=_dev()).add_(0.5).to(stored)
    dy = torch.rand(1, N, M, generator=g, device=_dev()).add_(0.5).to(dtype)
    if dtype == torch.float32:
        dy = dy.bfloat16().float()  # the leading piece alone: its sums are the long ones
    p = tsm.pack_activation(x)
    got = tsm.packed_weight_grad(dy if aligned else _offset(dy), p, dtype=torch.float32)
    rows, cols = torch.arange(0, M, 37, device=_dev()), torch.arange(0, D, 13, device=_dev())
    v = p.unpack(torch.float32)[0][:, cols].double()
    want = dy[0][:, rows].double().t() @ v
    pieces = 2 if dtype != stored or (dtype == torch.float16 and not aligned) else 1
    segment = 512 if dtype == torch.float32 else 2048
    tol = 1.1 * (pieces * (segment / 16 + 1) / 2 * 2.0 ** -23
                 + (N / segment + 1) / 2 * 2.0 ** -24)
    err = ((got[rows][:, cols].double() - want) / want).abs().max()
    assert err <= tol, (float(err), tol)


# ---------------------------------------------------------------------------
# rows that overlap or are one and the same
# ---------------------------------------------------------------------------
def _overlapping(g, B, T, D, dtype):
    """Windows of a signal (fewer and more positions than channels, by the
    caller), rows a step of four apart, one sequence or one position for all."""
    signal = _normal(g, B, T + D, dtype=dtype)
    yield "windows", signal.unfold(1, D, 1)[:, :T]
    yield "steps", _normal(g, B, 4 * T + D, dtype=dtype).unfold(1, D, 4)[:, :T]
    yield "batch", _normal(g, 1, T, D, dtype=dtype).expand(B, T, D)
    yield "time", _normal(g, B, 1, D, dtype=dtype).expand(B, T, D)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("B,T,D", [(3, 4, 10), (2, 70, 16), (2, 9, 64)])
def test_overlapping_rows_equal_their_copies(dtype, B, T, D):
    """Forward and backward of the recurrence and the norms on inputs whose rows
    overlap: what contiguous copies of them give (rows that are loaded in other
    units sum in another order: a few roundings)."""
    import torch_semimarkov_b200 as tsm

    g = _gen(T)
    w = [_normal(g, D, scale=0.2, shift=1.0) for _ in range(3)]
    dh, dn = _normal(g, B, T, D, dtype=dtype), _normal(g, B, T, D, dtype=dtype)
    u = ref.UNIT[dtype]

    def every(x):
        leaves = [x.detach().requires_grad_(True) for _ in range(2)]
        h, s = tsm.gated_linear_recurrence(*leaves)
        out = [h, s, *torch.autograd.grad((h, s), leaves, (dh, s.detach()))]
        leaves = [x.detach().requires_grad_(True) for _ in range(3)]
        r, n = tsm.gated_residual_norm(*leaves, *w)
        out += [r, n, *torch.autograd.grad((r, n), leaves, (dh, dn))]
        leaf = x.detach().requires_grad_(True)
        n = tsm.rms_norm(leaf, w[0])
        out += [n, *torch.autograd.grad(n, leaf, dn)]
        p = tsm.pack_activation(x)
        return out + [p.codes, p.scales, tsm.packed_weight_grad(x, p)]

    for how, x in _overlapping(g, B, T, D, dtype):
        for a, b in zip(every(x), every(x.contiguous())):
            if a.dtype in (torch.int8, torch.uint8):
                assert torch.equal(a, b), how
                continue
            a, b = a.detach().double(), b.detach().double()
            tol = 2 * u * b.abs() + 512 * ref.U32 * float(b.abs().max())
            assert ((a - b).abs() <= tol).all(), (how, float((a - b).abs().max()))


# ---------------------------------------------------------------------------
# padding of the encoder's features
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_encoder_padding_reaches_no_gradient(dtype, packed):
    """NaN and infinities past each length: outputs and every parameter's
    gradient are, bit for bit, those of zero padding."""
    import torch_semimarkov_b200 as tsm

    g = _gen(50)
    B, T, n = 3, 40, torch.tensor([40, 13, 0])
    live = ref.live_mask(n, B, T).to(_dev())[..., None]
    x, target = _normal(g, B, T, 7), _normal(g, B, T, 24)
    results = []
    for how in (0.0, float("nan"), float("inf")):
        torch.manual_seed(51)
        enc = tsm.GatedRecurrentEncoder(7, 24, checkpoint_8bit=packed, dtype=dtype).to(_dev())
        features = torch.where(live, x, torch.full_like(x, how)).requires_grad_(True)
        y = enc(features, n)
        (y.float() * target).sum().backward()
        results.append([y.detach(), features.grad, *(p.grad for p in enc.parameters())])
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.isfinite(b).all() and torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_encoder_padding_reaches_no_output_of_inference(dtype):
    import torch_semimarkov_b200 as tsm

    g = _gen(52)
    B, T, n = 3, 40, torch.tensor([40, 13, 0])
    live = ref.live_mask(n, B, T).to(_dev())[..., None]
    x = _normal(g, B, T, 7)
    enc = tsm.GatedRecurrentEncoder(7, 24, dtype=dtype).to(_dev())
    trained = enc(x, n).detach()
    with torch.no_grad():
        for how in (0.0, float("nan"), float("-inf")):
            y = enc(torch.where(live, x, torch.full_like(x, how)), n)
            assert torch.equal(y, trained) and not y[~live[..., 0]].any()


# ---------------------------------------------------------------------------
# gates at the ends of their types
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [37, 64, 512, 4100])
def test_norm_gates_at_their_limits(dtype, D):
    """silu is 0 at the lowest values of a type, as a masked gate has them, and
    far into saturation; its slope too.  Bounds as for any other gate."""
    from test_gpu_encoder_ops import _check_norm, _norm_inputs

    g = _gen(D)
    B, T = 2, 6
    t, w = _norm_inputs(g, B, T, D, dtype)
    low = torch.finfo(dtype).min
    values = torch.tensor([low, low / 2, low / 1e4, -2e4, -200.0, -128.0, -100.0, -88.0, -80.0, 0.0,
                           60.0, 200.0], device=_dev())
    pick = torch.randint(0, len(values), (B, T, D), generator=g, device=_dev())
    t["gate"] = values[pick].to(dtype)
    dr, dn = _normal(g, B, T, D, dtype=dtype), _normal(g, B, T, D, dtype=dtype)
    _check_norm(t, w, None, dr, dn)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_norm_gate_of_minus_infinity_closes_the_branch(dtype):
    import torch_semimarkov_b200 as tsm

    g = _gen(60)
    x, z = (_normal(g, 2, 5, 72, dtype=dtype) for _ in range(2))
    w = [torch.ones(72, device=_dev()) for _ in range(3)]
    leaves = [v.requires_grad_(True) for v in (x, z, torch.full_like(x, float("-inf")))]
    r, n = tsm.gated_residual_norm(*leaves, *w)
    assert torch.equal(r, x) and torch.equal(n, tsm.rms_norm(x, w[2]))
    _, gz, gg = torch.autograd.grad((r, n), leaves, (x.detach(), z.detach()))
    assert float(gz.abs().max()) <= 1e-30 and float(gg.abs().max()) <= 1e-30


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("at", [1, 3, 4, 8])
def test_checkpoints_at_any_place_of_a_buffer(dtype, at):
    """Codes and scales as slices of one byte buffer, as a file would hold them."""
    import torch_semimarkov_b200 as tsm

    g = _gen(70)
    x, dy = _normal(g, 2, 30, 72, dtype=dtype), _normal(g, 2, 30, 48, dtype=dtype)
    p = tsm.pack_activation(x)
    n = p.codes.numel()
    buffer = torch.zeros(at + n + p.scales.numel(), dtype=torch.uint8, device=_dev())
    codes = buffer[at:at + n].view(torch.int8).view(p.codes.shape)
    scales = buffer[at + n:].view(p.scales.shape)
    codes.copy_(p.codes), scales.copy_(p.scales)
    q = tsm.PackedActivation(codes, scales, p.channels, p.dtype)
    assert torch.equal(p.unpack(), q.unpack())
    assert torch.equal(tsm.packed_weight_grad(dy, p), tsm.packed_weight_grad(dy, q))
    w = _normal(g, 48, 72).requires_grad_(True)
    a, b = (torch.autograd.grad(tsm.packed_linear(x, w, packed=k), w, dy)[0] for k in (p, q))
    assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# infinite states
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("shift", [1.0, -30.0], ids=["gates near 0", "gates near -30"])
@pytest.mark.parametrize("B,T,D", [(1, 9000, 4), (64, 150, 512)],
                         ids=["segments", "one segment"])
def test_recurrence_infinities_pass_every_position(B, T, D, shift, reverse):
    """An infinite initial state, value or gradient stays infinite over any
    number of positions, however small the product of their gates, and however
    the positions are shared out: the formula's infinities, at its places."""
    from test_gpu_encoder_ops import _lam_max, _recurrence_bounds

    import torch_semimarkov_b200 as tsm

    g = _gen(T + D)
    inf = float("inf")
    gate = _normal(g, B, T, D, shift=shift)
    for what in ("state", "x", "grad"):
        x, s0, dh, ds = (_normal(g, B, T, D), _normal(g, B, D), _normal(g, B, T, D),
                         _normal(g, B, D))
        scale = [t.clone() for t in (x, s0, dh, ds)]
        if what == "state":
            s0[:, 0], s0[:, 1] = inf, -inf
        elif what == "x":
            x[:, T // 3, 0], x[:, T // 2, 1] = inf, -inf
        else:
            ds[:, 0], dh[:, T // 2, 1] = inf, -inf
        leaves = [t.requires_grad_(True) for t in (x, gate.clone(), s0)]
        h, s = tsm.gated_linear_recurrence(*leaves[:2], s0, reverse=reverse)
        got = (h, s, *torch.autograd.grad((h, s), leaves, (dh, ds)))
        want = ref.recurrence(x, gate, s0, None, reverse, dh, ds)
        tol = _recurrence_bounds(want, scale[0], scale[1], torch.float32, T,
                                 _lam_max(x, gate, None, reverse, scale[2], scale[3]))
        for v, k in zip(got, ("h", "state", "grad_x", "grad_gate", "grad_initial")):
            ref.assert_within(v, want[k], torch.nan_to_num(tol[k], posinf=0.0), f"{what}: {k}")


# ---------------------------------------------------------------------------
# forward-mode differentiation
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_tangents_are_refused_not_lost(grad_mode):
    """The operators have no forward-mode derivative; an input with a tangent is
    an error wherever it stands, whether or not it requires a gradient.  The plain
    product of packed_linear has one and keeps it."""
    import torch.autograd.forward_ad as fw

    import torch_semimarkov_b200 as tsm

    g = _gen(80)
    x, dy = _normal(g, 2, 9, 16), _normal(g, 2, 9, 16)
    w, s, wm = _normal(g, 16), _normal(g, 2, 16), _normal(g, 8, 16)
    p = tsm.pack_activation(x)
    with torch.set_grad_enabled(grad_mode), fw.dual_level():
        def dual(t):
            return fw.make_dual(t.clone(), torch.ones_like(t))

        calls = [lambda: tsm.gated_linear_recurrence(dual(x), x),
                 lambda: tsm.gated_linear_recurrence(x, dual(x)),
                 lambda: tsm.gated_linear_recurrence(x, x, dual(s)),
                 lambda: tsm.gated_linear_recurrence_step(dual(x[:, 0]), x[:, 0], s),
                 lambda: tsm.gated_linear_recurrence_step(x[:, 0], x[:, 0], dual(s)),
                 lambda: tsm.rms_norm(dual(x), w), lambda: tsm.rms_norm(x, dual(w)),
                 lambda: tsm.pack_activation(dual(x)),
                 lambda: tsm.packed_weight_grad(dual(dy), p)]
        for k in range(6):
            v = [x, x, x, w, w, w]
            v[k] = dual(v[k])
            calls.append(lambda v=tuple(v): tsm.gated_residual_norm(*v))
        for k, call in enumerate(calls):
            with pytest.raises(NotImplementedError):
                call()
        y = tsm.packed_linear(dual(x), wm)
        torch.testing.assert_close(fw.unpack_dual(y).tangent, torch.ones_like(x) @ wm.t())
        # without a tangent the calls are what they are outside
        h, _ = tsm.gated_linear_recurrence(x, x)
        n = tsm.rms_norm(x, w)
    assert torch.equal(h, tsm.gated_linear_recurrence(x, x)[0])
    assert torch.equal(n, tsm.rms_norm(x, w))


# ---------------------------------------------------------------------------
# packed_linear
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("trained", [True, False])
@pytest.mark.parametrize("how", ["rows", "slices", "time first"])
@pytest.mark.parametrize("dtype", TYPES[1:], ids=IDS[1:])
def test_packed_linear_rounds_once(dtype, how, trained):
    """Product and bias are rounded together: at most half a unit of the result
    (and 64 float32 steps of what is summed), not half a unit of the product more."""
    import torch_semimarkov_b200 as tsm

    g = _gen(90)
    B, T, D, M = 2, 200, 64, 96
    x = _normal(g, B, T, 3 * D, dtype=dtype)[..., D:2 * D]
    x = {"rows": x.contiguous(), "slices": x, "time first": x.transpose(0, 1).contiguous()
         .transpose(0, 1)}[how]
    w = _normal(g, M, D, scale=D ** -0.5, dtype=dtype).requires_grad_(trained)
    b = _normal(g, M, dtype=dtype).requires_grad_(trained)
    y = tsm.packed_linear(x, w, b).detach().double()
    assert y.shape == (B, T, M)
    xd, wd, bd = (t.detach().double() for t in (x, w, b))
    want = xd @ wd.t() + bd
    tol = ref.UNIT[dtype] * want.abs() + (D + 1) * ref.U32 * (xd.abs() @ wd.abs().t() + bd.abs())
    assert ((y - want).abs() <= tol + ref.TINY[dtype]).all()


def test_packed_linear_without_positions():
    import torch_semimarkov_b200 as tsm

    w = torch.ones(3, 8, device=_dev(), requires_grad=True)
    b = torch.ones(3, device=_dev(), requires_grad=True)
    for shape in ((0, 5, 8), (2, 0, 8)):
        x = torch.empty(shape, device=_dev(), requires_grad=True)
        y = tsm.packed_linear(x, w, b)
        assert y.shape == (*shape[:2], 3)
        for v in torch.autograd.grad(y.sum(), (x, w, b)):
            assert not v.any()
