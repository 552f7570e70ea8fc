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
