"""CPU-only checks of the encoder operators: refusals before any CUDA call,
size queries, and the float64 forms that the GPU tests compare with."""

import ctypes

import pytest
import torch

import encoder_reference as ref


def _recurrence(**kw):
    from torch_semimarkov_b200 import _lib

    base = dict(batch=0, T=10, D=4, dtype=0, reverse=0)
    base.update(kw)
    return ctypes.byref(_lib.SemicrfRecurrence(**base))


def _norm(**kw):
    from torch_semimarkov_b200 import _lib

    base = dict(batch=0, T=10, D=4, dtype=1, eps=1e-6, next_weight=1)
    base.update(kw)
    return ctypes.byref(_lib.SemicrfBlockNorm(**base))


def test_recurrence_validation_codes():
    from torch_semimarkov_b200 import _lib

    lib = _lib.load()

    def forward(p):
        return lib.semicrf_recurrence_forward(p, None, None, None, None, 0, None)

    assert forward(_recurrence()) == _lib.SEMICRF_OK  # no sequences: nothing to do
    assert forward(_recurrence(T=-1)) == _lib.SEMICRF_ERR_INVALID_ARGUMENT
    assert forward(_recurrence(D=0)) == _lib.SEMICRF_ERR_INVALID_ARGUMENT
    assert forward(_recurrence(dtype=3)) == _lib.SEMICRF_ERR_INVALID_ARGUMENT
    assert forward(_recurrence(batch=2)) == _lib.SEMICRF_ERR_INVALID_ARGUMENT  # null outputs
    assert forward(_recurrence(batch=1 << 20, T=1 << 30)) == _lib.SEMICRF_ERR_UNSUPPORTED
    assert lib.semicrf_recurrence_saved_size(_recurrence(batch=2, T=1000, D=8)) >= 4 * 2 * 15 * 8
    assert lib.semicrf_recurrence_saved_size(_recurrence(D=0)) == 0
    assert lib.semicrf_recurrence_step(2, 4, 0, None, 0, None, 0, None, None, None, None,
                                       None) == _lib.SEMICRF_ERR_INVALID_ARGUMENT


def test_block_norm_validation_codes():
    from torch_semimarkov_b200 import _lib

    lib = _lib.load()

    def forward(p, codes=None):
        seq = ctypes.byref(_lib.SemicrfSequence(1, 0, 0))
        return lib.semicrf_block_norm_forward(p, seq, seq, None, codes, None, None)

    assert forward(_norm()) == _lib.SEMICRF_OK
    assert forward(_norm(D=9000)) == _lib.SEMICRF_ERR_UNSUPPORTED
    assert forward(_norm(eps=-1.0)) == _lib.SEMICRF_ERR_INVALID_ARGUMENT
    assert forward(_norm(eps=float("nan"))) == _lib.SEMICRF_ERR_INVALID_ARGUMENT
    assert forward(_norm(next_weight=None)) == _lib.SEMICRF_ERR_INVALID_ARGUMENT
    some = _lib.SemicrfSequence(1, 40, 4)
    assert forward(_norm(batch=2)) == _lib.SEMICRF_ERR_INVALID_ARGUMENT
    # a branch needs its gate and weights; codes need scales
    assert forward(_norm(batch=2, residual=some, branch=some)) == \
        _lib.SEMICRF_ERR_INVALID_ARGUMENT
    assert forward(_norm(batch=2, residual=some), codes=1) == _lib.SEMICRF_ERR_INVALID_ARGUMENT


def test_pack_validation_codes():
    from torch_semimarkov_b200 import _lib

    lib = _lib.load()
    seq = ctypes.byref(_lib.SemicrfSequence(None, 0, 0))
    assert lib.semicrf_pack(0, 5, 8, 1, seq, None, None, None, None) == _lib.SEMICRF_OK
    assert lib.semicrf_pack(2, 5, 8, 1, seq, None, None, None, None) == \
        _lib.SEMICRF_ERR_INVALID_ARGUMENT
    assert lib.semicrf_pack(2, 5, 8, 9, seq, None, None, None, None) == \
        _lib.SEMICRF_ERR_INVALID_ARGUMENT
    assert lib.semicrf_unpack(0, 8, 1, None, None, None, None) == _lib.SEMICRF_OK
    assert lib.semicrf_unpack(3, 8, 1, None, None, None, None) == \
        _lib.SEMICRF_ERR_INVALID_ARGUMENT
    assert lib.semicrf_packed_weight_grad_workspace_size(2, 5, 8, 0, 1) == 0
    assert lib.semicrf_packed_weight_grad(2, 5, 8, 3, 1, seq, None, None, 1, None, 0, None, None, 0,
                                          None) == _lib.SEMICRF_ERR_INVALID_ARGUMENT


def test_cpu_tensors_raise():
    import torch_semimarkov_b200 as tsm

    x, w = torch.zeros(1, 3, 4), torch.ones(4)
    for call in (lambda: tsm.gated_linear_recurrence(x, x),
                 lambda: tsm.gated_linear_recurrence_step(x[0], x[0], x[0]),
                 lambda: tsm.gated_residual_norm(x, x, x, w, w, w),
                 lambda: tsm.rms_norm(x, w),
                 lambda: tsm.pack_activation(x),
                 lambda: tsm.packed_linear(x, torch.zeros(2, 4)),
                 lambda: tsm.PackedActivation(torch.zeros(1, 3, 32, dtype=torch.int8),
                                              torch.zeros(1, 3, 1, dtype=torch.uint8), 4,
                                              torch.float32).unpack()):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="batch, time, channel"):
        tsm.gated_linear_recurrence(x[0], x[0])


def test_lengths_are_checked_on_the_host():
    from torch_semimarkov_b200 import _lib

    dev = torch.device("cpu")
    assert _lib.valid_lengths(None, 2, 5, dev) is None
    assert _lib.valid_lengths([5, 0], 2, 5, dev).dtype == torch.int64
    for bad in ([6, 0], [-1, 2], [1], [1.0, 2.0]):
        with pytest.raises(ValueError, match="lengths"):
            _lib.valid_lengths(bad, 2, 5, dev)


def test_struct_mirrors_match_the_header():
    """Field order and sizes: two pointers-and-strides triples and the scalars."""
    from torch_semimarkov_b200 import _lib

    assert ctypes.sizeof(_lib.SemicrfSequence) == 24
    for mirror, packed in ((_lib.SemicrfSequence, _lib._SEQUENCE),
                           (_lib.SemicrfRecurrence, _lib._RECURRENCE),
                           (_lib.SemicrfBlockNorm, _lib._BLOCK_NORM)):
        assert ctypes.sizeof(mirror) == packed.size
    p = _lib.SemicrfBlockNorm(1, 2, 3, 1, 0.5, (4, 5, 6), (7, 8, 9), (10, 11, 12), 13, 14, 15, 16)
    assert bytes(p) == _lib._BLOCK_NORM.pack(1, 2, 3, 1, 0.5, *range(4, 17))
    p = _lib.SemicrfRecurrence(1, 2, 3, 2, 1, (4, 5, 6), (7, 8, 9), 10, 11)
    assert bytes(p) == _lib._RECURRENCE.pack(1, 2, 3, 2, 1, *range(4, 12))
    assert ctypes.sizeof(_lib.SemicrfRecurrence) == 3 * 8 + 8 + 2 * 24 + 16
    assert ctypes.sizeof(_lib.SemicrfBlockNorm) == 3 * 8 + 8 + 3 * 24 + 4 * 8


def test_reference_recurrence_gradient_by_differentiation():
    g = torch.Generator().manual_seed(0)
    B, T, D = 2, 6, 3
    n = torch.tensor([6, 4])
    x, gate = (torch.randn(B, T, D, generator=g, dtype=torch.float64).requires_grad_(True)
               for _ in range(2))
    s0 = torch.randn(B, D, generator=g, dtype=torch.float64).requires_grad_(True)
    dh = torch.randn(B, T, D, generator=g, dtype=torch.float64)
    ds = torch.randn(B, D, generator=g, dtype=torch.float64)
    for reverse in (False, True):
        s, rows = s0, [None] * T
        for t in (range(T - 1, -1, -1) if reverse else range(T)):
            f = torch.sigmoid(gate[:, t])
            live = (t < n)[:, None]
            s = torch.where(live, f * s + (1 - f) * x[:, t], s)
            rows[t] = torch.where(live, s, torch.zeros_like(s))
        grads = torch.autograd.grad((torch.stack(rows, 1), s), (x, gate, s0), (dh, ds))
        want = ref.recurrence(x, gate, s0, n, reverse, dh, ds)
        for v, k in zip(grads, ("grad_x", "grad_gate", "grad_initial")):
            torch.testing.assert_close(v, want[k], rtol=1e-11, atol=1e-12)


def test_reference_checkpoint_step():
    """No scale could be halved, and no code passes 127."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(1, 50, 32, generator=g) * torch.exp(3 * torch.randn(1, 50, 1, generator=g))
    codes, byte, values = ref.stored(x, None)
    top = codes.abs().amax(-1)
    assert int(top.max()) <= 127 and int(top.min()) >= 63
    assert ((values - x).abs() <= 0.5 * torch.exp2(byte.double() - 127)).all()


def test_encoder_arguments():
    import torch_semimarkov_b200 as tsm

    with pytest.raises(ValueError, match="num_layers"):
        tsm.GatedRecurrentEncoder(4, 8, num_layers=0)
    with pytest.raises(ValueError, match="dtype"):
        tsm.GatedRecurrentEncoder(4, 8, dtype=torch.float64)
    enc = tsm.GatedRecurrentEncoder(4, 8, num_layers=3)
    assert len(enc.initial_states(2)) == 3 and enc.initial_states(2)[0].shape == (2, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        enc(torch.zeros(1, 3, 4))
