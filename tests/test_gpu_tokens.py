"""The modules of tt_rsl_rl_amd.tokens on the GPU: TokenEmbedding under autograd, AdamW as a torch optimiser, and the example
that runs them with the loss."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_embedding_gradient(cuda, dtype):
    """Against torch's indexing in fp32: whole numbers, whose sums are exact."""
    from tt_rsl_rl_amd.tokens import TokenEmbedding

    torch.manual_seed(0)
    embed = TokenEmbedding(50, 24, scale=2.0, device=cuda, dtype=dtype)
    with torch.no_grad():
        embed.weight.copy_(torch.randint(-4, 5, (50, 24)))
    tokens = torch.randint(0, 50, (6, 7), device=cuda)
    tokens[0, 0] = -1
    d = torch.randint(-2, 3, (6, 7, 24), device=cuda).to(dtype)
    out = embed(tokens)
    assert out.shape == (6, 7, 24) and out.dtype == dtype
    out.backward(d)
    table = embed.weight.detach().float().requires_grad_()
    want = table[tokens.clamp(min=0)] * 2.0 * (tokens >= 0)[..., None]
    want.backward(d.float())
    assert torch.equal(out.float(), want) and torch.equal(embed.weight.grad.float(), table.grad)
    embed.weight.grad = None
    embed(tokens).float().sum().backward()  # a gradient that is a broadcast scalar
    assert float(embed.weight.grad.float().sum()) == 41 * 24 * 2.0


def _params(cuda, dtype):
    g = torch.Generator().manual_seed(1)
    return [torch.nn.Parameter(torch.randn(*s, generator=g).to(device=cuda, dtype=dtype)) for s in ((33, 17), (300,), (5, 4, 3))]


def test_adamw_matches_torch_over_steps(cuda):
    """fp32, two groups, one parameter without a gradient at first: torch.optim.AdamW after clip_grad_norm_ (the same operations in
    fp32 but for the order of the norm's sum)."""
    from tt_rsl_rl_amd.tokens import AdamW

    ours, theirs = _params(cuda, torch.float32), _params(cuda, torch.float32)
    groups = lambda p: [dict(params=p[:1], weight_decay=0.1), dict(params=p[1:], lr=3e-3, weight_decay=0.0)]  # noqa: E731
    a, b = AdamW(groups(ours), lr=1e-3, max_grad_norm=0.7), torch.optim.AdamW(groups(theirs), lr=1e-3, foreach=False)
    g = torch.Generator().manual_seed(2)
    for step in range(5):
        for i, (p, q) in enumerate(zip(ours, theirs)):
            if i == 1 and step < 2:
                continue
            p.grad = torch.randn(*p.shape, generator=g).to(cuda)
            q.grad = p.grad.clone()
        norm = torch.nn.utils.clip_grad_norm_([q for q in theirs if q.grad is not None], 0.7)
        a.step()
        b.step()
        assert abs(float(a.norm[0]) - float(norm)) < 1e-5 * float(norm)
    for p, q in zip(ours, theirs):
        assert (p - q).abs().max() <= 2e-6 * (1 + q.abs().max())
        assert a.state[p]["step"] == int(b.state[q]["step"])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_adamw_state_round_trip(cuda, bits, dtype, tmp_path):
    """Saved and loaded between steps: the same bits as without."""
    from tt_rsl_rl_amd.tokens import AdamW

    def run(reload):
        p = _params(cuda, dtype)
        opt = AdamW(p, lr=1e-2, max_grad_norm=1.0, state_bits=bits)
        g = torch.Generator().manual_seed(3)
        for step in range(4):
            if reload and step == 2:
                torch.save(opt.state_dict(), tmp_path / "opt.pt")
                opt = AdamW(p, lr=1e-2, max_grad_norm=1.0, state_bits=bits)
                opt.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
                with pytest.raises(ValueError, match="state_bits"):
                    AdamW(p, state_bits=40 - bits).load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
            for q in p:
                q.grad = torch.randn(*q.shape, generator=g).to(device=cuda, dtype=dtype)
            opt.step()
        return [q.detach() for q in p]

    for x, y in zip(run(False), run(True)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_mixed_types(cuda, bits):
    """fp32 and bf16 parameters in one optimiser, with and without masters: what each gets alone."""
    from tt_rsl_rl_amd.tokens import AdamW

    for masters in (True, False):
        together = [_params(cuda, torch.float32)[0], _params(cuda, torch.bfloat16)[1], _params(cuda, torch.float32)[2]]
        alone = [torch.nn.Parameter(p.detach().clone()) for p in together]
        opt, each = AdamW(together, lr=1e-2, state_bits=bits, masters=masters), [AdamW([p], lr=1e-2, state_bits=bits, masters=masters) for p in alone]
        g = torch.Generator().manual_seed(4)
        for _ in range(3):
            for p, q in zip(together, alone):
                p.grad = torch.randn(*p.shape, generator=g).to(device=cuda, dtype=p.dtype)
                q.grad = p.grad.clone()
            opt.step()
            for o in each:
                o.step()
        for p, q in zip(together, alone):
            assert torch.equal(p, q)


def test_example_learns(cuda):
    spec = importlib.util.spec_from_file_location("token_policy", ROOT / "examples" / "token_policy.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    for bits in (32, 8):
        history = example.train(iterations=25, state_bits=bits)
        assert history[0] < 0.1 and history[-1] > 0.5, history
