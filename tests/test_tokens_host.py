"""tt_rsl_rl_amd.tokens without a GPU: constructor checks, and that CPU tensors are refused."""

from __future__ import annotations

import pytest
import torch


def test_constructors_check_their_arguments():
    from tt_rsl_rl_amd.tokens import AdamW, TokenEmbedding

    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(state_bits=16),
                dict(max_grad_norm=0.0)):
        with pytest.raises(ValueError, match="AdamW"):
            AdamW(p, **bad)
    with pytest.raises(ValueError, match="scale"):
        TokenEmbedding(4, 2, scale=0.0)
    embed = TokenEmbedding(1000, 64, scale=8.0)
    assert abs(float(embed.weight.std()) * 8.0 - 1.0) < 0.02


def test_cpu_tensors_are_refused_and_counts_stay():
    from tt_rsl_rl_amd.tokens import AdamW, TokenEmbedding

    with pytest.raises(ValueError, match="GPU"):
        TokenEmbedding(4, 2)(torch.zeros(3, dtype=torch.int64))
    p = torch.nn.Parameter(torch.zeros(3))
    opt = AdamW([p])
    opt.step()  # nothing has a gradient
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="GPU"):
        opt.step()
    assert opt.state[p]["step"] == 0
