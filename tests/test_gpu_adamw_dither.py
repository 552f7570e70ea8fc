"""AdamW's 8-bit states over many steps: codes rounded by chance keep the value they stand for on average, so that the moments
follow the gradients as 32-bit ones do."""

from __future__ import annotations

import pytest
import torch

from tests import token_reference as ref

pytestmark = pytest.mark.gpu


def _step(ops, g, step, state, dither=True, b1=0.9, b2=0.999, lr=0.0):
    qm, qv, sm, sv = state
    p = torch.zeros_like(g)
    ops.adamw_step([p], [g], [qm], [qv], step=step, lr=lr, beta1=b1, beta2=b2, scales=([sm], [sv]), dither=dither)
    return p


def _zero(n, cuda):
    blocks = -(-n // 256)
    return (torch.zeros(n, dtype=torch.int8, device=cuda), torch.zeros(n, dtype=torch.uint8, device=cuda), torch.zeros(blocks, device=cuda),
            torch.zeros(blocks, device=cuda))


def test_codes_keep_the_value_on_average(cuda):
    """From the zero state with one gradient, for the numbers of 4,000 steps: each code is one of the value's two neighbours, and
    their mean is the value to six deviations of such a mean (and 20 draws' weight where the deviation is near 0).  m = 0.1 g and
    v = 0.001 g^2 over four decades; in fp32 to 1e-5 of a block's largest code's distance, 2.4e-7 of the value each."""
    from tt_rsl_rl_amd import ops

    n, draws = 1000, 4000
    g = torch.Generator().manual_seed(0)
    x = 10.0 ** (-4 * torch.rand(n, generator=g)) * torch.where(torch.rand(n, generator=g) < 0.5, -1.0, 1.0)
    x[::256] = 1.0
    x[5], x[6] = 0.0, 1e-7
    x = x.to(cuda)
    state = _zero(n, cuda)
    sum_m, sum_v = (torch.zeros(n, dtype=torch.float64, device=cuda) for _ in range(2))
    for step in range(1, draws + 1):
        for t in state:
            t.zero_()
        _step(ops, x, step, state)
        cm, cv = state[0].double(), state[1].double()
        dm = (cm / 127).square() * cm.sign()
        dv = (cv / 255) ** 4
        sum_m, sum_v = sum_m + dm, sum_v + dv
        if step == 1:
            low_m, high_m, low_v, high_v = cm.abs(), cm.abs(), cv, cv
        low_m, high_m = torch.minimum(low_m, cm.abs()), torch.maximum(high_m, cm.abs())
        low_v, high_v = torch.minimum(low_v, cv), torch.maximum(high_v, cv)
    for want, got, low, high, top, power in ((x.double(), sum_m / draws, low_m, high_m, 127, 2),
                                             (x.double().square(), sum_v / draws, low_v, high_v, 255, 4)):
        k = torch.floor(want.abs() ** (1 / power) * top * (1 - 1e-9)).clamp(max=top - 1)
        below, above = (k / top) ** power, ((k + 1) / top) ** power
        p = ((want.abs() - below) / (above - below)).clamp(0, 1)
        # a value within 1e-4 of a code's may be taken for one on its other side
        assert bool(((low >= k - (p < 1e-4).double()) & (high <= k + 1 + (p > 1 - 1e-4).double()))[want.abs() > 1e-9].all())
        bound = (above - below) * (6 * (p * (1 - p) / draws).sqrt() + 20 / draws + 1e-5) + 2.4e-7 * want.abs()
        keep = want.abs() > 1e-9 if power == 4 else want.abs() >= 0  # (below, v is held at the first code)
        assert bool(((got - want).abs() <= bound)[keep].all())
    assert int(high_v[5]) == 0 and int(high_m[5]) == 0  # 0 stays 0
    assert int(low_v[6]) == 1 and int(high_v[6]) == 1  # and v, however small, is not


def test_codes_go_by_the_step_alone(cuda):
    from tt_rsl_rl_amd import ops

    x = torch.randn(70000, generator=torch.Generator().manual_seed(1)).to(cuda)
    states = [_zero(x.numel(), cuda) for _ in range(4)]
    for state, step, dither in zip(states, (7, 7, 8, 7), (True, True, True, False)):
        _step(ops, x, step, state, dither=dither)
    for a, b in zip(states[0], states[1]):
        assert torch.equal(a, b)
    for a, b in zip(states[0][2:], states[2][2:]):  # the scales are the largest values, without chance
        assert torch.equal(a, b)
    for i in (0, 1):
        assert 0.2 < float((states[0][i] != states[2][i]).float().mean()) < 0.6  # (both draws of a code up or down: a third differ)
        assert int((states[0][i].int() - states[3][i].int()).abs().max()) == 1
    up_m, up_v = (states[0][i].int().abs() - states[2][i].int().abs() for i in (0, 1))
    both = torch.stack([up_m.float(), up_v.float()])
    assert abs(float(torch.corrcoef(both)[0, 1])) < 5 / 70000**0.5  # m's chance is not v's
    assert abs(float(torch.corrcoef(torch.stack([both[0, 1:], both[0, :-1]]))[0, 1])) < 5 / 70000**0.5  # nor the next element's


def _train(cuda, gradient, steps, **options):
    """Three optimisers of one parameter each, on the same gradients: 32 bits, 8 bits, and 8 bits rounded to nearest."""
    from tt_rsl_rl_amd import ops
    from tt_rsl_rl_amd.tokens import AdamW

    n, lr = 64 * 256, 1e-3
    g = torch.Generator(device=cuda).manual_seed(0)
    params = [torch.nn.Parameter(torch.zeros(n, device=cuda)) for _ in range(2)]
    opts = [AdamW([p], lr=lr, weight_decay=0.0, state_bits=b) for p, b in zip(params, (32, 8))]
    nearest, state = torch.zeros(n, device=cuda), _zero(n, cuda)
    seen = []
    for step in range(1, steps + 1):
        grad = gradient(step, torch.randn(n, generator=g, device=cuda))
        for p, o in zip(params, opts):
            p.grad = grad
            o.step()
        ops.adamw_step([nearest], [grad], [state[0]], [state[1]], step=step, lr=lr, weight_decay=0.0, scales=([state[2]], [state[3]]))
        if step in (500, steps):
            seen.append([p.detach().clone() for p in (*params, nearest)])
    wide, narrow = opts[0].state[params[0]], opts[1].state[params[1]]
    v = [wide["exp_avg_sq"].double(), ref.decode_v(narrow["exp_avg_sq"].cpu(), narrow["exp_avg_sq_scale"].cpu()).to(cuda),
         ref.decode_v(state[1].cpu(), state[3].cpu()).to(cuda)]
    return v, seen


def test_second_moment_follows_gradients_that_shrink(cuda):
    """Half of each block's gradients a tenth from step 1,000 on, 5,000 steps more.  The codes' values are kept on average, so the
    mean ratio of the two v is 1; a code lies 5 % from the next at a hundredth of the largest v, and draws of 500 steps' changes
    of 0.1 % leave a deviation of sqrt(0.05 * 0.001 * 500) = 0.16: 0.002 for the mean of 8,192, ten of which are allowed."""
    first = torch.arange(64 * 256, device=cuda) % 256 < 128

    def gradient(step, noise):
        return torch.where(first, noise * 0.1, noise) if step > 1000 else noise

    v, _ = _train(cuda, gradient, 6000)
    for part in (first, ~first):
        assert abs(float((v[1] / v[0])[part].mean()) - 1) < 0.02
    assert float((v[2] / v[0])[first].mean()) > 10  # (what the header says of codes rounded to nearest)


def test_small_gradients_move_parameters_as_in_32_bits(cuda):
    """A quarter of each block has a constant gradient, a hundredth of the others' deviation, for 500 steps, then none for 5,000.
    Where v is 16 % off by chance (above; here a code is 16 % and 1 / sqrt(v) larger by 3 / 8 of the variance, 3 %), parameters
    move as far as in 32 bits to a tenth, and then no further than they do."""
    small = torch.arange(64 * 256, device=cuda) % 256 < 64

    def gradient(step, noise):
        return torch.where(small, torch.full_like(noise, 0.01 if step <= 500 else 0.0), noise)

    _, seen = _train(cuda, gradient, 5500)
    moved = [float(p[small].mean()) for p in seen[0]]
    after = [float((b - a)[small].mean()) for a, b in zip(*seen)]
    assert abs(moved[1] / moved[0] - 1) < 0.1, moved
    assert abs(after[1] - after[0]) < 3e-3, after  # 3 steps of 1e-3
    assert abs(after[2] - after[0]) > 0.05, after  # (to nearest: momentum that never ends)
