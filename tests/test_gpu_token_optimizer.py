"""tokens.AdamW on the GPU as an optimiser of torch's: copies, schedulers, parameters that come twice."""

from __future__ import annotations

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_parameter_that_comes_twice_is_refused(cuda):
    from tt_rsl_rl_amd import ops
    from tt_rsl_rl_amd.tokens import AdamW

    x = [torch.ones(300, device=cuda) for _ in range(40)]
    g, m, v = ([torch.ones(300, device=cuda) for _ in range(41)] for _ in range(3))
    with pytest.raises(ValueError, match=r"adamw_step: params\[40\] comes a second time"):
        ops.adamw_step([*x, x[7]], g, m, v, step=1, lr=0.1)
    assert all(float(t.min()) == 1.0 for t in x)
    empty = torch.ones(0, device=cuda)
    ops.adamw_step([empty, empty], [empty, empty], [empty, empty], [empty, empty], step=1, lr=0.1)
    p = torch.nn.Parameter(torch.ones(5, device=cuda))
    p.grad = torch.ones_like(p)
    with pytest.warns(UserWarning, match="duplicate"):
        opt = AdamW([p, p])
    with pytest.raises(ValueError, match="second time"):
        opt.step()
    assert float(p.min()) == 1.0 and opt.state[p]["step"] == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_a_copy_goes_on_with_the_same_bits(cuda, bits):
    from tt_rsl_rl_amd.tokens import AdamW

    g = torch.Generator().manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(n, generator=g).to(device=cuda, dtype=d)) for n, d in ((700, torch.float32), (300, torch.bfloat16))]
    opt = AdamW(params, lr=1e-2, betas=(0.8, 0.95), max_grad_norm=1.0, state_bits=bits)
    schedule = torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=1e-2, total_steps=10)

    def step(o, seed):
        h = torch.Generator().manual_seed(seed)
        for group in o.param_groups:
            for p in group["params"]:
                p.grad = torch.randn(*p.shape, generator=h).to(device=cuda, dtype=p.dtype)
        o.step()

    for i in range(3):
        step(opt, i)
        schedule.step()
    other = copy.deepcopy(opt)
    for i in (5, 6):
        step(opt, i)
        step(other, i)
    for p, q in zip(params, other.param_groups[0]["params"]):
        assert p.data_ptr() != q.data_ptr() and torch.equal(p, q)
    assert torch.equal(opt.norm, other.norm)
