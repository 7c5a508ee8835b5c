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
