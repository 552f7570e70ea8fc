"""What the token operators write is marked as written: a backward pass that has kept one of the tensors refuses to go on, as after
torch's own in-place operations."""

from __future__ import annotations

import pytest
import torch


def test_the_mark():
    from tt_rsl_rl_amd import _lib

    written = _lib.tensor_table().written
    a, b, c = torch.zeros(2), torch.zeros(2, requires_grad=True), torch.zeros(2)
    written(a, [b.detach(), None], (c,), None)
    assert (a._version, b._version, c._version) == (1, 1, 1)
    written(torch.nn.ParameterList([torch.nn.Parameter(torch.zeros(1))]), [])
    with torch.inference_mode():
        d = torch.zeros(2)
    written(d, a)
    assert a._version == 2
    for bad in (3, [a, "x"]):
        with pytest.raises(TypeError):
            written(bad)
    y = (b * b).sum()
    written(b.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
def test_a_graph_from_before_the_step_is_refused(cuda):
    from tt_rsl_rl_amd.tokens import AdamW

    layer = torch.nn.Linear(4, 4, bias=False, device=cuda)
    opt = AdamW(layer.parameters(), max_grad_norm=1.0)
    x = torch.randn(3, 4, device=cuda, requires_grad=True)
    kept = layer(x).sum()
    layer(x).square().sum().backward()
    state_version = [layer.weight._version]
    opt.step()
    state = opt.state[layer.weight]
    assert layer.weight._version == state_version[0] + 1 and state["exp_avg"]._version == 1 and opt.norm._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()


@pytest.mark.gpu
def test_outputs_are_marked(cuda):
    from tt_rsl_rl_amd import ops

    rows, vocab = 5, 40
    tok = torch.arange(rows, device=cuda)
    old, adv, stats = torch.zeros(rows, device=cuda), torch.ones(rows, device=cuda), torch.empty(8, device=cuda)
    scores = torch.randn(rows, vocab, device=cuda, requires_grad=True)
    logits = torch.tanh(scores)  # whose backward pass reads its output
    lp, h = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
    ops.token_log_probs(logits.detach(), tok, lp, h)
    assert (lp._version, h._version, logits._version) == (1, 1, 0)
    apart = torch.empty_like(logits)
    ops.token_ppo_loss(logits.detach(), tok, old, adv, apart, stats, logp=lp)
    assert (apart._version, stats._version, lp._version, logits._version) == (1, 1, 2, 0)
    ops.token_ppo_loss(logits.detach(), tok, old, adv, logits.detach(), stats)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        logits.backward(apart)
    table, out = torch.randn(vocab, 8, device=cuda), torch.empty(rows, 8, device=cuda)
    ops.embedding_fwd(tok, table, out)
    ops.embedding_bwd(tok, out, table)
    assert (out._version, table._version) == (1, 1)
    with pytest.raises(ValueError):
        ops.embedding_fwd(tok, table, out[:2])
    assert out._version == 1
