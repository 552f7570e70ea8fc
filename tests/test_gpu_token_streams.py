"""The token operators on a stream of the caller's: their inputs become right on it, late, and nothing orders another stream behind
it, so that a launch on any other one would read what was there before."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_token_ops import BF16, OUT, _all_ops, _all_state, _ops

pytestmark = pytest.mark.gpu

INPUTS = ("tok", "table", "x", "old", "adv", "mask", "m", "v")


def _late(cuda, inputs, run):
    """run() on another stream behind a few ms of work and the copies that make the inputs right; wrong ones (rows in another
    order, all of them in range) until then."""
    right = {k: t.clone() for k, t in inputs.items()}
    for t in inputs.values():
        t.copy_(t.flip(0))
    big = torch.ones(4096, 4096, device=cuda)
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        for _ in range(40):
            big = torch.mm(big, big).clamp_(-1.0, 1.0)
        for k, t in inputs.items():
            t.copy_(right[k])
        run()
    pending = not other.query()
    torch.cuda.synchronize()
    return pending


@pytest.mark.parametrize("rows,vocab,dim", [(6000, 700, 96), (20_000, 700, 96), (40, 20_011, 64)])
def test_all_on_another_stream(cuda, rows, vocab, dim):
    ops = _ops()
    a, b = (_all_state(cuda, ops, rows=rows, vocab=vocab, dim=dim) for _ in range(2))
    _all_ops(ops, a)
    assert _late(cuda, {k: b[k] for k in INPUTS}, lambda: _all_ops(ops, b)), "the delay has to outlast the launches"
    for k in OUT:
        assert torch.equal(a[k], b[k]), k


def test_modules_on_another_stream(cuda):
    """TokenEmbedding's backward pass and AdamW's step, with scratch memory of their own."""
    from tt_rsl_rl_amd.tokens import AdamW, TokenEmbedding

    def make():
        torch.manual_seed(0)
        embed = TokenEmbedding(500, 64, scale=2.0, device=cuda, dtype=BF16)
        return embed, AdamW(embed.parameters(), lr=1e-2, max_grad_norm=1.0, state_bits=8)

    def run(embed, opt, tok, d):
        for _ in range(2):
            opt.zero_grad(set_to_none=True)
            embed(tok).backward(d)
            opt.step()

    g = torch.Generator(device=cuda).manual_seed(1)
    tok, d = torch.randint(0, 500, (15_000,), generator=g, device=cuda), torch.randn(15_000, 64, generator=g, device=cuda).to(BF16)
    one, two = make(), make()
    run(*one, tok, d)
    run(*make(), tok, d)  # (every lazy set-up has happened)
    assert _late(cuda, dict(tok=tok, d=d, weight=two[0].weight.data), lambda: run(*two, tok, d))
    assert torch.equal(one[0].weight, two[0].weight) and torch.equal(one[1].norm, two[1].norm)
