"""GatedRecurrentEncoder: the operators together, and with the CRF head."""

import pytest
import torch

import encoder_reference as ref

pytestmark = pytest.mark.gpu


def _dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _encoder(seed, **kw):
    import torch_semimarkov_b200 as tsm

    torch.manual_seed(seed)
    return tsm.GatedRecurrentEncoder(**kw).to(_dev())


def _plain(enc, features, lengths):
    """The encoder's formulas, position by position, in float64 on the CPU."""
    w = {k: v.detach().cpu().double() for k, v in enc.state_dict().items()}
    B, T = features.shape[:2]
    live = ref.live_mask(lengths, B, T)
    r = features.cpu().double() @ w["embed.weight"].t() + w["embed.bias"]
    n = ref.block_norm(r, None, None, None, None, w["first_weight"], lengths, enc.eps)["n"]
    for k in range(enc.num_layers):
        p = n @ w[f"in_weight.{k}"].t() + w[f"in_bias.{k}"]
        v, f, o = p.split(enc.hidden_dim, dim=-1)
        h = ref.recurrence(v, f, None, lengths, enc.bidirectional and k % 2 == 1)["h"]
        out = ref.block_norm(r, h, o, w[f"branch_weight.{k}"], w[f"residual_scale.{k}"],
                             w[f"next_weight.{k}"], lengths, enc.eps)
        r, n = out["r"], out["n"]
    return torch.where(live[..., None], n, torch.zeros_like(n))


# Three blocks of norms (outputs of order 1): each block rounds its stream,
# projections and normed values to the type once or twice, so about 8 roundings
# a block reach an output, in float32 with the products' 64-term sums beside.
@pytest.mark.parametrize("dtype,tol", [(torch.float32, 3 * 64 * 2.0 ** -24 * 8),
                                       (torch.bfloat16, 3 * 8 * 2.0 ** -8)],
                         ids=["fp32", "bf16"])
@pytest.mark.parametrize("bidirectional", [True, False])
def test_encoder_forward(dtype, tol, bidirectional):
    enc = _encoder(0, input_dim=9, hidden_dim=64, num_layers=3, bidirectional=bidirectional,
                   dtype=dtype)
    g = torch.Generator(device=_dev()).manual_seed(1)
    x = torch.randn(3, 70, 9, generator=g, device=_dev()).to(dtype).float()
    n = torch.tensor([70, 41, 0])
    precise = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        with torch.no_grad():
            got = enc(x, n)
            kept = enc(x, n.to(_dev()))
    finally:
        torch.backends.cuda.matmul.allow_tf32 = precise
    want = _plain(enc, x, n)
    assert got.dtype == dtype and torch.equal(got, kept)
    err = (got.cpu().double() - want).abs().max()
    assert err <= tol * max(1.0, float(want.abs().max())), float(err)
    assert torch.equal(got[2], torch.zeros_like(got[2]))


def test_encoder_gradients_with_8bit_checkpoints():
    """float32 activations: gradients through the checkpoints differ from those
    without only by the projections' stored inputs, each off by at most half of
    2^e with max <= 127 * 2^e, less than 1 / 127 of its group's largest."""
    g = torch.Generator(device=_dev()).manual_seed(2)
    x = torch.randn(2, 60, 8, generator=g, device=_dev())
    n = torch.tensor([60, 23])
    target = torch.randn(2, 60, 48, generator=g, device=_dev())
    grads = {}
    for packed in (True, False):
        enc = _encoder(3, input_dim=8, hidden_dim=48, num_layers=2, checkpoint_8bit=packed,
                       dtype=torch.float32)
        ((enc(x, n) - target).square().mean()).backward()
        grads[packed] = {k: p.grad for k, p in enc.named_parameters()}
    for k, exact in grads[False].items():
        off = (grads[True][k] - exact).norm() / exact.norm()
        # only weights whose input is stored may differ at all beyond float32 rounding
        assert off <= (1.0 / 127 if k.startswith("in_weight") else 1e-5), (k, float(off))
        assert torch.isfinite(exact).all()


def test_encoder_step_matches_forward():
    enc = _encoder(4, input_dim=6, hidden_dim=40, num_layers=2, bidirectional=False,
                   dtype=torch.float32)
    g = torch.Generator(device=_dev()).manual_seed(5)
    x = torch.randn(3, 20, 6, generator=g, device=_dev())
    with torch.no_grad():
        want = enc(x)
    states = enc.initial_states(3)
    for t in range(20):
        torch.testing.assert_close(enc.step(x[:, t], states), want[:, t], rtol=1e-4, atol=1e-4)
    with pytest.raises(ValueError, match="bidirectional"):
        _encoder(4, input_dim=6, hidden_dim=8).step(x[:, 0], states)
    with pytest.raises(ValueError, match="states"):
        enc.step(x[:, 0], states[:1])


def test_checkpoints_hold_a_quarter_of_the_projection_inputs():
    """What the backward keeps: in 8 bits the projections' inputs take
    (1 + 1/32) / 4 of their float32 size."""
    held = {}
    for packed in (True, False):
        enc = _encoder(6, input_dim=8, hidden_dim=64, num_layers=2, checkpoint_8bit=packed,
                       dtype=torch.float32)
        x = torch.randn(2, 500, 8, device=_dev())
        seen = {}

        def keep(t):
            seen[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
            return t

        with torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
            y = enc(x)
        held[packed] = sum(seen.values())
        y.sum().backward()
    one = 2 * 500 * 64 * 4
    saved = held[False] - held[True]
    assert saved >= 2 * one * (1 - (1 + 1 / 32) / 4) - 4096, (held, one)


def test_encoder_and_head_learn_segments():
    """A few steps on sequences whose labels are runs: the loss falls, and the
    decoded segmentation covers each sequence."""
    import torch_semimarkov_b200 as tsm

    torch.manual_seed(7)
    dev = _dev()
    B, T, C, F = 4, 120, 3, 5
    labels = (torch.arange(T, device=dev)[None] // 10 + torch.arange(B, device=dev)[:, None]) % C
    features = torch.nn.functional.one_hot(labels, F).float() + 0.3 * torch.randn(B, T, F,
                                                                                 device=dev)
    lengths = torch.tensor([120, 90, 50, 20], device=dev)
    enc = tsm.GatedRecurrentEncoder(F, 64, num_layers=2).to(dev)
    head = tsm.SemiMarkovCRFHead(C, 16, hidden_dim=64).to(dev)
    opt = torch.optim.Adam([*enc.parameters(), *head.parameters()], lr=3e-3)
    losses = []
    for _ in range(30):
        opt.zero_grad()
        loss = head.compute_loss(enc(features, lengths).float(), lengths, labels)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.5 * losses[0], losses
    for p in enc.parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all()
    with torch.no_grad():
        result = head.decode_with_traceback(enc(features, lengths).float(), lengths)
    for b, segments in enumerate(result.segments):
        assert segments[0].start == 0 and segments[-1].end == int(lengths[b]) - 1
