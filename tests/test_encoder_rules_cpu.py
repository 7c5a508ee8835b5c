"""CPU-only checks of rules that the encoder operators share: the layout of what
the kernels write, what they refuse, what a lost copy leaves behind."""

import pytest
import torch


def _windows(B, T, D):
    """Every window of D values of a signal: neighbouring rows overlap."""
    return torch.arange(float(B * (T + D - 1))).view(B, T + D - 1).unfold(1, D, 1)


@pytest.mark.parametrize("B,T,D", [(3, 4, 10), (3, 10, 4), (4, 6, 8), (1, 5, 7), (2, 5, 1)])
def test_outputs_have_contiguous_channels_whatever_the_inputs_rows_do(B, T, D):
    """The kernels write rows with channel stride 1 from the batch and time
    strides that they are given; no two rows of an output may meet."""
    from torch_semimarkov_b200 import _lib

    dense = torch.zeros(B, T, D)
    wide = torch.zeros(B, T, 3 * D + 1)
    for t in (_windows(B, T, D), dense, dense.transpose(0, 1), wide[..., 1:D + 1],
              dense[:1].expand(B, T, D), dense[:, :1].expand(B, T, D),
              torch.zeros(B + 8 * T + D).as_strided((B, T, D), (1, 8, 1))):
        out = _lib.rows_like(t)
        assert out.shape == t.shape and out.dtype == t.dtype
        seen = set()
        sb, st, _ = out.stride()
        for b in range(t.shape[0]):
            for k in range(t.shape[1]):
                seen.update(range(b * sb + k * st, b * sb + k * st + t.shape[2]))
                if D > 1:
                    assert out.stride(2) == 1
        assert len(seen) == t.numel()
        assert max(seen) < out.untyped_storage().nbytes() // 4
    # an order of its own is kept
    assert _lib.rows_like(dense.transpose(0, 1)).stride() == dense.transpose(0, 1).stride()


def test_misaligned_addresses_are_refused_before_any_launch():
    """Codes are read 8 at a time, activations by their elements; an address
    between them is an error code, not a launch."""
    import ctypes

    from torch_semimarkov_b200 import _lib

    lib, bad = _lib.load(), _lib.SEMICRF_ERR_INVALID_ARGUMENT
    good = ctypes.byref(_lib.SemicrfSequence(64, 40, 8))
    odd = ctypes.byref(_lib.SemicrfSequence(65, 40, 8))
    for at in (1025, 1026, 1028):
        assert lib.semicrf_pack(2, 5, 8, 1, good, None, at, 4096, None) == bad
        assert lib.semicrf_unpack(3, 8, 1, at, 4096, 8192, None) == bad
        assert lib.semicrf_packed_weight_grad(2, 5, 8, 3, 1, good, at, 4096, 1, None, 0, 8192, 4096,
                                              1 << 30, None) == bad
        p = ctypes.byref(_lib.SemicrfBlockNorm(2, 5, 8, 1, 0.0, (64, 40, 8), (0, 0, 0), (0, 0, 0),
                                               None, None, 64, None))
        none = ctypes.byref(_lib.SemicrfSequence(None, 0, 0))
        assert lib.semicrf_block_norm_forward(p, none, good, None, at, 4096, None) == bad
    assert lib.semicrf_pack(2, 5, 8, 1, odd, None, 1024, 4096, None) == bad
    p = ctypes.byref(_lib.SemicrfRecurrence(2, 5, 8, 1, 0, (65, 40, 8), (64, 40, 8), None, None))
    assert lib.semicrf_recurrence_forward(p, good, 64, None, 64, 1 << 30, None) == bad


def test_codes_at_an_odd_place_of_a_buffer_are_copied():
    from torch_semimarkov_b200 import _lib

    buffer = torch.arange(1 + 64, dtype=torch.int8)
    codes = buffer[1:].view(1, 2, 32)
    assert codes.data_ptr() % 8 != 0 and codes.is_contiguous()
    kept = _lib.aligned_codes(codes)
    assert kept.data_ptr() % 8 == 0 and torch.equal(kept, codes)
    assert _lib.aligned_codes(kept) is kept


def _walk_with_marks(marked_f, marked_d):
    """The recurrence's chunk as its computing warps walk it (8 warps of 8
    positions, compositions handed on between them) for 4 channels, on inputs that
    look valid, with the marks of a chunk that never came."""
    g = torch.Generator().manual_seed(0)
    warps, run, C = 8, 8, 4
    f, x, d = (torch.rand(warps, run, C, generator=g) for _ in range(3))
    n = 1 - f
    nan = float("nan")
    f[:, 0, marked_f] = nan
    d[:, run - 1, marked_d] = nan
    P, S, M = torch.ones(warps, C), torch.zeros(warps, C), torch.zeros(warps, C)
    for i in range(run):
        P, S = f[:, i] * P, f[:, i] * S + n[:, i] * x[:, i]
    for i in reversed(range(run)):
        M = f[:, i] * (d[:, i] + M)
    h, dx, dg = (torch.empty(warps, run, C) for _ in range(3))
    for w in range(warps):
        state, mu = torch.ones(C), torch.ones(C)
        for k in range(w):
            state = P[k] * state + S[k]
        for k in reversed(range(w + 1, warps)):
            mu = P[k] * mu + M[k]
        before = torch.empty(run, C)
        for i in range(run):
            before[i] = state
            state = f[w, i] * state + n[w, i] * x[w, i]
            h[w, i] = state
        for i in reversed(range(run)):
            lam = d[w, i] + mu
            mu = f[w, i] * lam
            dx[w, i] = lam * n[w, i]
            dg[w, i] = mu * n[w, i] * (before[i] - x[w, i])
    return h, dx, dg


def test_marks_of_a_lost_chunk_reach_every_value():
    """All channels of a lane have to be marked, and in the backward both ends of
    a run; then no state and no gradient of the chunk is a number."""
    every, none, one = slice(None), slice(0, 0), slice(0, 1)
    h, dx, dg = _walk_with_marks(every, every)
    assert torch.isnan(h).all() and torch.isnan(dx).all() and torch.isnan(dg).all()
    h, dx, dg = _walk_with_marks(one, none)  # a mark on one channel leaves the others
    assert not torch.isnan(h[..., 1:]).any() and not torch.isnan(dx).all()
    h, dx, dg = _walk_with_marks(every, none)  # the state's marks alone miss dx
    assert torch.isnan(h).all() and not torch.isnan(dx).all()


def test_every_wait_for_a_chunk_marks_all_channels():
    """In the recurrence's kernels: whatever waits for a chunk marks what comes
    of it with mark_lost, and nothing marks half a pair."""
    import os
    import re

    here = os.path.dirname(os.path.abspath(__file__))
    with open(os.path.join(here, "..", "torch_semimarkov_b200", "csrc", "recurrence.cu")) as file:
        source = file.read()
    waits = [m.start() for m in re.finditer(r"if \(ok\) ok = barrier_wait\(&full", source)]
    assert len(waits) == 3
    for at, end in zip(waits, waits[1:] + [len(source)]):
        failed = source[source.index("if (!ok)", at, end):end]
        assert "mark_lost(" in failed[:120]
    assert not re.search(r"\.[xy] = __uint_as_float\(0x7fc00000u\)", source)
    assert "mark_lost(f[0]), mark_lost(d[kRun - 1])" in source
