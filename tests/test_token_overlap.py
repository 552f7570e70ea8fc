"""Outputs that lie on inputs: one block would write what another has yet to read, so the token operators refuse them, before any
HIP call.  (Addresses here are numbers; nothing is read from them.)"""

from __future__ import annotations

import ctypes

import pytest

M = 1 << 20  # memory of an operand's own


def _embedding(entry, **more):
    from tt_rsl_rl_amd import _lib as L

    L.load()
    d = dict(tokens=1 * M, src=2 * M, ld_src=8, dst=3 * M, ld_dst=8, count=4, vocab=10, dim=8, scale=1.0)
    args = ctypes.byref(L.EmbeddingArgs(**{**d, **more}))
    L.call(entry, *((args, None) if entry.endswith("fwd") else (args, 4 * M, 1 << 18, None)))


def _loss(entry, **more):
    from tt_rsl_rl_amd import _lib as L

    d = dict(logits=1 * M, ld_logits=10, tokens=2 * M, mask=3 * M, old_logp=4 * M, ref_logp=5 * M, advantages=6 * M, d_logits=7 * M, ld_d_logits=10,
             logp=8 * M, entropy=9 * M, stats=10 * M, rows=4, vocab=10, clip_low=0.2, clip_high=0.2, temperature=1.0)
    L.call(entry, ctypes.byref(L.TokenLossArgs(**{**d, **more})), 11 * M, 1 << 18, None)


@pytest.mark.parametrize("entry,src,dst", [("ppo_embedding_fwd", 10, 4), ("ppo_embedding_bwd", 4, 10)])
def test_embedding(entry, src, dst):
    for more in (dict(dst=2 * M), dict(dst=2 * M + src * 32 - 4), dict(dst=2 * M - dst * 32 + 4), dict(dst=1 * M), dict(dst=1 * M + 28),
                 dict(ld_src=16, ld_dst=16, dst=2 * M + 28), dict(ld_src=16, ld_dst=24, dst=2 * M + 32)):
        with pytest.raises(ValueError, match="overlap"):
            _embedding(entry, **more)


def test_loss():
    vectors = dict(tokens=2, mask=3, old_logp=4, ref_logp=5, advantages=6)
    for out in ("logp", "entropy", "stats", "d_logits"):
        for at in vectors.values():
            with pytest.raises(ValueError, match="overlap"):
                _loss("ppo_token_ppo_loss", **{out: at * M})
    for more in (dict(logp=9 * M), dict(stats=8 * M + 12), dict(entropy=7 * M + 8), dict(logp=1 * M), dict(d_logits=1 * M + 4), dict(d_logits=1 * M - 4),
                 dict(ld_logits=20, ld_d_logits=20, d_logits=1 * M + 36), dict(ld_logits=20, ld_d_logits=30, d_logits=1 * M + 40)):
        with pytest.raises(ValueError, match="overlap"):
            _loss("ppo_token_ppo_loss", **more)
    for more in (dict(logp=2 * M), dict(entropy=3 * M), dict(logp=9 * M), dict(entropy=1 * M)):
        with pytest.raises(ValueError, match="overlap"):
            _loss("ppo_token_log_probs", **more)


@pytest.mark.gpu
def test_columns_side_by_side_are_taken(cuda):
    """Views of one matrix that share its rows and no column."""
    import torch

    from tt_rsl_rl_amd import ops

    g = torch.Generator().manual_seed(0)
    both = torch.randn(6, 50, generator=g).to(cuda)
    tok, old, adv = torch.arange(6, device=cuda), torch.full((6,), -3.0, device=cuda), torch.ones(6, device=cuda)
    want, stats, again = torch.empty(6, 25, device=cuda), torch.empty(8, device=cuda), torch.empty(8, device=cuda)
    ops.token_ppo_loss(both[:, :25].contiguous(), tok, old, adv, want, stats)
    ops.token_ppo_loss(both[:, :25], tok, old, adv, both[:, 25:], again)
    assert torch.equal(both[:, 25:], want) and torch.equal(stats, again)
    ops.embedding_fwd(tok, both[:, :20], both[:, 20:40], scale=2.0)
    assert torch.equal(both[:, 20:40], both[:, :20] * 2)
    ops.token_log_probs(both[:, :25], tok, old, None)
    with pytest.raises(ValueError, match="overlap"):
        ops.token_ppo_loss(both[:, :25], tok, old, adv, None, stats, logp=old)
