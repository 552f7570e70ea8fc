"""What the functions of tt_rsl_rl_amd.tokens between embedding and logits ask of the operators, on the CPU (the operators are stood in for)."""

from __future__ import annotations

import pytest
import torch

from tt_rsl_rl_amd import ops, tokens


@pytest.fixture
def asked(monkeypatch):
    """The gradients that each call of ops.linear_cross_entropy is asked for; it gives a loss of 2 and gradients of ones."""
    calls = []

    def stand_in(hidden, weight, tok, d_hidden, d_weight, stats, mask=None, temperature=1.0, denom=None):
        calls.append((d_hidden is not None, d_weight is not None))
        stats.fill_(2.0)
        for d in (d_hidden, d_weight):
            if d is not None:
                d.fill_(1.0)

    monkeypatch.setattr(ops, "linear_cross_entropy", stand_in)
    return calls


def test_no_gradients_are_made_where_none_can_be_asked_for(asked):
    hidden, tok = torch.randn(3, 4), torch.zeros(3, dtype=torch.int64)
    weight = torch.nn.Parameter(torch.randn(5, 4))
    with torch.no_grad():
        loss = tokens.linear_cross_entropy(hidden, weight, tok)
    assert float(loss) == 2.0 and not loss.requires_grad
    with torch.inference_mode():
        tokens.linear_cross_entropy(hidden.clone().requires_grad_(), weight, tok)
    tokens.linear_cross_entropy(hidden, weight.detach(), tok)
    assert asked == [(False, False)] * 3


def test_gradients_are_made_of_what_needs_them(asked):
    hidden, tok = torch.randn(3, 4), torch.zeros(3, dtype=torch.int64)
    weight = torch.nn.Parameter(torch.randn(5, 4))
    tokens.linear_cross_entropy(hidden, weight, tok).mul(0.5).backward()
    assert torch.equal(weight.grad, torch.full((5, 4), 0.5))
    leaf = hidden.clone().requires_grad_()
    tokens.linear_cross_entropy(leaf, weight.detach(), tok).backward()
    assert torch.equal(leaf.grad, torch.ones(3, 4))
    tokens.linear_cross_entropy(leaf, weight, tok)
    assert asked == [(False, True), (True, False), (True, True)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients_are_multiplied_by_the_losses_factor_in_float32(monkeypatch, dtype):
    """And rounded once: 0.1 is none of the 16-bit types' values."""
    g = torch.Generator().manual_seed(0)
    made = torch.randn(7, 4, generator=g).to(dtype), torch.randn(50, 4, generator=g).to(dtype)

    def stand_in(hidden, weight, tok, d_hidden, d_weight, stats, mask=None, temperature=1.0, denom=None):
        stats.fill_(2.0), d_hidden.copy_(made[0]), d_weight.copy_(made[1])

    monkeypatch.setattr(ops, "linear_cross_entropy", stand_in)
    hidden, weight = (torch.zeros_like(m).requires_grad_() for m in made)
    (tokens.linear_cross_entropy(hidden, weight, torch.zeros(7, dtype=torch.int64)) * 0.1).backward()
    for x, m in zip((hidden, weight), made):
        assert x.grad.dtype is dtype and torch.equal(x.grad, (m.float() * torch.tensor(0.1)).to(dtype))


@pytest.mark.gpu
def test_the_backward_pass_makes_no_copies(cuda):
    """What it allocates at its height is the gradients themselves (and what the allocator rounds up)."""
    g = torch.Generator(device=cuda).manual_seed(1)
    hidden = torch.randn(64, 512, generator=g, device=cuda).to(torch.bfloat16).requires_grad_()
    weight = torch.randn(20000, 512, generator=g, device=cuda).to(torch.bfloat16).requires_grad_()
    loss = tokens.linear_cross_entropy(hidden, weight, torch.randint(0, 20000, (64,), generator=g, device=cuda)) * 3.0
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    loss.backward()
    assert torch.cuda.max_memory_allocated() - before <= 2 * (hidden.numel() + weight.numel()) + (4 << 20)


@pytest.mark.parametrize("packed", [False, True])
def test_only_tokens_of_no_sequence_are_cleared(monkeypatch, packed):
    """One sequence of all tokens has none: its outputs and gradients are all written by the operators."""
    cleared = []
    zeros = torch.Tensor.new_zeros
    monkeypatch.setattr(torch.Tensor, "new_zeros", lambda self, *shape, **more: cleared.append(shape) or zeros(self, *shape, **more))
    monkeypatch.setattr(ops, "decay_attention_fwd", lambda q, k, v, log_decay, out, **more: out.fill_(1.0))
    monkeypatch.setattr(ops, "decay_attention_bwd", lambda g, q, k, v, log_decay, *grads, **more: [x.fill_(1.0) for x in grads] and None)
    q, k, v = (torch.zeros(6, heads, 4, requires_grad=True) for heads in (2, 1, 1))
    out, _ = tokens.decay_attention(q, k, v, torch.zeros(1), cu_seqlens=torch.tensor([0, 5]) if packed else None)
    out.sum().backward()
    assert len(cleared) == (4 if packed else 0) and all(bool((x.grad == 1).all()) for x in (q, k, v))
