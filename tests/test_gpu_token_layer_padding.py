"""Tokens of no sequence in tokens.decay_attention and tokens.DecayMixer: padding before the first sequence and behind the last one."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_token_ops import BF16, F32, U

pytestmark = pytest.mark.gpu


def _leave_nan_behind(cuda, *shapes, dtype=F32):
    """What is allocated next, of these sizes, holds NaN."""
    kept = [torch.full(shape, float("nan"), dtype=dtype, device=cuda) for shape in shapes for _ in range(20)]
    del kept


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_outputs_of_no_sequence_are_zeros(cuda, dtype):
    from tt_rsl_rl_amd.tokens import decay_attention

    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(90, heads, 16, generator=g).to(dtype).to(cuda).requires_grad_() for heads in (4, 2, 2))
    ld, cu = torch.tensor([-0.1, -0.01], device=cuda), torch.tensor([7, 40, 40, 77], device=cuda)
    _leave_nan_behind(cuda, (90, 4, 16), dtype=dtype)
    out, _ = decay_attention(q, k, v, ld, cu_seqlens=cu)
    assert not bool(out[:7].any()) and not bool(out[77:].any()) and bool(out.isfinite().all())
    out.float().square().sum().backward()
    for x in (q, k, v):
        assert not bool(x.grad[:7].any()) and not bool(x.grad[77:].any()) and bool(x.grad[7:77].any())


def test_padding_leaves_a_layers_gradients_alone(cuda):
    """Every parameter's gradient is that of the same tokens without padding, whatever memory held before.  Both are fp32 sums over 70 tokens (of padding, zeros) of
    products whose operands have gone through sums of up to 64 terms twice: 300 U of the largest such sum over magnitudes, taken to be 30 times the largest result."""
    from tt_rsl_rl_amd.tokens import DecayMixer

    torch.manual_seed(2)
    layer = DecayMixer(64, 4, 2, 16, device=cuda)
    g = torch.Generator().manual_seed(3)
    x, weight = torch.randn(90, 64, generator=g).to(cuda), torch.randn(90, 64, generator=g).to(cuda)
    weight[:7], weight[77:] = 0, 0  # (the loss does not look at padding)
    positions = torch.arange(90, device=cuda)
    cu = torch.tensor([7, 40, 77], device=cuda)

    def gradients(lo, hi):
        layer.zero_grad(set_to_none=True)
        _leave_nan_behind(cuda, (hi - lo, 4, 16), (hi - lo, 2, 16), (hi - lo, 64), (hi - lo, 128))
        y, _ = layer(x[lo:hi], positions[lo:hi], cu - lo)
        (y * weight[lo:hi]).sum().backward()
        return {n: p.grad.clone() for n, p in layer.named_parameters()}

    padded, alone = gradients(0, 90), gradients(7, 77)
    for name, want in alone.items():
        assert bool(padded[name].isfinite().all()), name
        assert (padded[name] - want).abs().max() <= 300 * 30 * U * want.abs().max(), name
