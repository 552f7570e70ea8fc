"""Plain 64-bit forms of the token operators, on the CPU: what tests/test_gpu_token_ops.py compares the kernels with, and
tests/test_token_reference.py checks by itself (against autograd and differences)."""

from __future__ import annotations

import torch


def embedding(tokens: torch.Tensor, table: torch.Tensor, scale: float) -> torch.Tensor:
    t = tokens.reshape(-1).long()
    ok = (t >= 0) & (t < table.shape[0])
    rows = table.double()[t.clamp(0, table.shape[0] - 1)] * scale
    return torch.where(ok[:, None], rows, torch.zeros_like(rows))


def embedding_grad(tokens: torch.Tensor, d_out: torch.Tensor, vocab: int, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """The table's gradient, and the sums of its summands' magnitudes (what a bound on rounding is in terms of)."""
    t = tokens.reshape(-1).long()
    ok = (t >= 0) & (t < vocab)
    x = d_out.double()[ok] * scale
    out = torch.zeros(vocab, d_out.shape[1], dtype=torch.float64)
    return out.index_add(0, t[ok], x), out.index_add(0, t[ok], x.abs())


def rows_that_count(tokens: torch.Tensor, vocab: int, mask: torch.Tensor | None) -> torch.Tensor:
    ok = (tokens >= 0) & (tokens < vocab)
    return ok if mask is None else ok & (mask != 0)


def token_loss(logits, tokens, old_logp, advantages, ref_logp=None, mask=None, clip=(0.2, 0.2), kl_coef=0.0, entropy_coef=0.0,
               temperature=1.0, denom=None) -> dict:
    """logp, entropy, stats and d_logits by the formulas, with no automatic derivative."""
    rows, vocab = logits.shape
    counts = rows_that_count(tokens, vocab, mask)
    n = float(denom) if denom is not None else float(counts.sum())
    z = logits.double() / temperature
    live = counts & ~((z == -float("inf")).all(1))
    out = {"logp": torch.zeros(rows, dtype=torch.float64), "entropy": torch.zeros(rows, dtype=torch.float64),
           "d_logits": torch.zeros(rows, vocab, dtype=torch.float64)}
    terms = torch.zeros(5, dtype=torch.float64)
    for r in live.nonzero()[:, 0].tolist():
        t = int(tokens[r])
        m = z[r].max()
        e = torch.exp(z[r] - m)
        log_p = z[r] - m - torch.log(e.sum())
        p = e / e.sum()
        log_p0 = torch.where(p > 0, log_p, torch.zeros_like(log_p)) if not torch.isnan(p).any() else log_p
        h = -(p * log_p0).sum()
        lp = log_p[t]
        ratio = torch.exp(lp - float(old_logp[r]))
        adv = float(advantages[r])
        first, second = -adv * ratio, -adv * ratio.clamp(1 - clip[0], 1 + clip[1])
        g = first if bool(first >= second) else torch.zeros_like(first)
        kl = torch.zeros_like(lp)
        if ref_logp is not None:
            d = float(ref_logp[r]) - lp
            kl = torch.exp(d) - d - 1
            g = g + kl_coef * (1 - torch.exp(d))
        row = -g * p + entropy_coef * p * (log_p0 + h)
        row[t] += g
        out["d_logits"][r] = row / (n * temperature)
        out["logp"][r], out["entropy"][r] = lp, h
        outside = (ratio < 1 - clip[0]) | (ratio > 1 + clip[1])
        terms += torch.stack([torch.maximum(first, second), kl, h, outside.double(), float(old_logp[r]) - lp])
    mean = terms / n if bool(counts.any()) else torch.zeros_like(terms)
    loss = mean[0] + kl_coef * mean[1] - entropy_coef * mean[2]
    out["stats"] = torch.cat([loss[None], mean])
    return out


def adamw(p, g, m, v, step, lr, beta1, beta2, eps, weight_decay, clip_coef=1.0):
    """One AdamW step in 64 bits: the new p, m, v."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * clip_coef
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    m_hat, v_hat = m / (1 - beta1**step), v / (1 - beta2**step)
    return p - lr * weight_decay * p - lr * m_hat / (v_hat.sqrt() + eps), m, v


BLOCK = 256


def _blocks(x: torch.Tensor) -> torch.Tensor:
    n = x.numel()
    return torch.nn.functional.pad(x.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)


def decode_m(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    f = _blocks(q.double())
    return (f.sign() * scale.double()[:, None] * (f.abs() / 127) ** 2).view(-1)[: q.numel()]


def decode_v(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return (scale.double()[:, None] * (_blocks(q.double()) / 255) ** 4).view(-1)[: q.numel()]
